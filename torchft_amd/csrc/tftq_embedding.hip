// Rows of a table by number, scaled, and the gradient of the table.
//
//    y[t] = scale table[ids[t]];   dtable[v] = scale (the sum of dy[t] over the t with ids[t] = v)
//
// A number outside the table has a row of zeros and no gradient (a rank that holds a part of a vocabulary
// looks up its own part, and the ranks' rows are summed); so it never reads out of range.
//
// The gradient is a sum over sorted tokens (tftq_sort.h), fp32, in an order that ids alone decide.  The sorted
// tokens are cut into chunks of equal size, so that a token that half of the text consists of is no longer to work on
// than any other: a team sums a chunk's runs, writes the table's row where a run begins and ends inside the
// chunk, and leaves fp32 sums where it goes on outside (at most one at each end).  A second launch adds up the sums of
// runs over several chunks.  The rows of no token are zeros, most of the memory that is written: the whole table is
// filled while the tokens are sorted, on the compute units that the sort leaves idle.  To leave out the rows that have tokens, and to fill the
// others beside the chunks, took 222 us for 128256 rows of 8 KB and 8192 tokens, against this way's 202.
#include "tftq_sort.h"

struct EmbeddingArgs {
    uint64_t ids, table, out;
    int64_t stride;  // bytes from row to row of the table
    int64_t row0, rows;
    int64_t vocab;
    int cols, wide;
    float scale;
};

// Bound by memory: 8192 tokens of 4096 bf16 17.5 us where their rows are in the last-level cache (7.7 TB/s), 26 where not.
template <class T, int TEAM, int U, bool NARROW>
__global__ __launch_bounds__(256) void k_embedding(const EmbeddingArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM;
    const int lane = threadIdx.x % TEAM;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (row >= a.rows) return;
    const int64_t id = a.wide ? as_global<const int64_t>(a.ids)[row] : as_global<const int32_t>(a.ids)[row];
    const bool inside = id >= 0 && id < a.vocab;
    const float scale = inside ? a.scale : 0.0f;  // zeros outside, whatever the scale
    const uint64_t from = a.table + (uint64_t)(id * a.stride), to = a.out + (uint64_t)(row * a.cols) * ESZ;
    for (int col = lane * EPV; col < a.cols; col += U * TEAM * EPV) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            Piece p = piece_of<EPV, NARROW>(col + u * TEAM * EPV, a.cols);
            p.in = p.in && inside;
            raw[u] = load_row<ESZ, NARROW, false>(from, p, a.cols);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float f[EPV];
            Elem<T>::unpack(raw[u], f);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] *= scale;
            store_row<ESZ, NARROW>(to, piece_of<EPV, NARROW>(col + u * TEAM * EPV, a.cols), a.cols, Elem<T>::pack(f));
        }
    }
}

struct TableArgs {
    uint64_t dy, keys, order, heads, tails, dtable;  // heads, tails: fp32 [chunks][sums_stride(cols)]
    int64_t n, chunks, vocab, first;  // the launch's first workgroup of the first columns
    int cols, chunk, across;          // tokens of a chunk, teams across the columns
    float scale;
};

// A lane sums the columns of one vector over a chunk of CHUNK tokens; neighbouring workgroups are `across` parts of the
// same chunks.  The chunk's tokens are read into LDS first: then every row's address is known, and U rows are on their way at once.
// 8192 tokens of 4096 bf16 20.6 us (68 MB read, 38 written: 5.1 TB/s), 4096 of 2048 8.2.
template <class T, int TEAM, int CHUNK, bool NARROW>
__global__ __launch_bounds__(256) void k_embedding_backward(const TableArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, U = 16;
    constexpr u32 NONE = 0xFFFFFFFFu;
    __shared__ u32 keys[TEAMS * CHUNK + 2], order[TEAMS * CHUNK];  // and the neighbours' keys
    const int part = (int)(blockIdx.x % (u32)a.across);
    const int64_t chunk0 = (a.first + blockIdx.x / (u32)a.across) * TEAMS, first = chunk0 * CHUNK;
    for (int i = threadIdx.x; i < TEAMS * CHUNK + 2; i += 256) {
        const int64_t at = first + i - 1;
        keys[i] = at >= 0 && at < a.n ? as_global<const u32>(a.keys)[at] : NONE;
    }
    for (int i = threadIdx.x; i < TEAMS * CHUNK; i += 256)
        if (first + i < a.n) order[i] = min(as_global<const u32>(a.order)[first + i], (u32)a.n - 1);  // whatever memory says
    __syncthreads();
    const int team = TEAM == 64 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64) : (int)threadIdx.x / TEAM;
    const int64_t chunk = chunk0 + team;
    const Piece piece = piece_of<EPV, NARROW>((part * TEAM + (int)threadIdx.x % TEAM) * EPV, a.cols);
    if (chunk >= a.chunks || !piece.in) return;
    const u32 *key = keys + 1 + team * CHUNK, *from = order + team * CHUNK;
    const u32 previous = key[-1], next = key[CHUNK];
    float acc[EPV] = {};
    u32 current = NONE;

    auto leave = [&](bool last) {  // the run of `current` ends, or the chunk does
        if (current >= (u32)a.vocab) return;
        if (current == previous || (last && next == current)) {
            store_sums((current == previous ? a.heads : a.tails) + (uint64_t)(chunk * sums_stride(a.cols)) * 4, piece, acc);
            return;
        }
        float f[EPV];
#pragma unroll
        for (int i = 0; i < EPV; i++) f[i] = acc[i] * a.scale;
        store_row<ESZ, NARROW, false>(a.dtable + (uint64_t)current * (uint64_t)a.cols * ESZ, piece, a.cols, Elem<T>::pack(f));
    };
#pragma unroll 1
    for (int at = 0; at < CHUNK; at += U) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            raw[u] = u32x4{0, 0, 0, 0};
            if (key[at + u] < (u32)a.vocab) raw[u] = load_row<ESZ, NARROW>(a.dy + (uint64_t)from[at + u] * (uint64_t)a.cols * ESZ, piece, a.cols);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const u32 k = key[at + u];
            if (k != current) {
                leave(false);
                current = k;
#pragma unroll
                for (int i = 0; i < EPV; i++) acc[i] = 0.0f;
            }
            float f[EPV];
            Elem<T>::unpack(raw[u], f);
#pragma unroll
            for (int i = 0; i < EPV; i++) acc[i] += f[i];
        }
    }
    leave(true);
}

// How many of n sorted keys are not above k, by a wavefront: 64 probes at once.
DEV int64_t first_above(const GLOBAL u32 *keys, int64_t n, u32 k)
{
    const int lane = threadIdx.x & 63;
    int64_t lo = 0;
    while (n > 0) {  // the answer is in lo to lo + n
        const int64_t step = (n + 63) >> 6, at = (int64_t)lane * step + step - 1;
        const int count = __builtin_popcountll(__ballot(at < n && keys[lo + at] <= k));  // a run of lanes from the first on
        lo += count * step;
        n = min(n - count * step, step - 1);
    }
    return lo;
}

// The runs of several chunks: a workgroup to the chunk where one begins and TEAM vectors of columns; its teams
// share the chunks, and add up in their order.  Most find no run that begins: 5.5 us for 8192 tokens of 4096 bf16, of which 6 %
// are the same.
template <class T, int TEAM, bool NARROW>
__global__ __launch_bounds__(256) void k_embedding_join(const TableArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM;
    __shared__ float add[TEAMS][TEAM][EPV + 1];
    const int64_t chunk = a.first + blockIdx.x / (u32)a.across, begin = chunk * a.chunk, end = begin + a.chunk;
    if (end >= a.n) return;
    const GLOBAL u32 *keys = as_global<const u32>(a.keys);
    const u32 before = keys[begin > 0 ? begin - 1 : 0], first = keys[begin], key = keys[end - 1], next = keys[end];
    if (key >= (u32)a.vocab || next != key) return;                   // no run goes on
    if (begin > 0 && first == key && before == key) return;          // it began before
    // the chunks that begin with the key: 64 looked at together, or else as the sorted numbers that they are
    const int64_t ahead = (chunk + 1 + (threadIdx.x & 63)) * a.chunk;
    const uint64_t others = ~__ballot(ahead < a.n && keys[ahead] == key);
    int64_t count = 1 + (others ? __builtin_ctzll(others) : 64);
    if (!others) count += (first_above(keys + (chunk + 65) * a.chunk, a.n - (chunk + 65) * a.chunk, key) + a.chunk - 1) / a.chunk;
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const Piece piece = piece_of<EPV, NARROW>(((int)(blockIdx.x % (u32)a.across) * TEAM + lane) * EPV, a.cols);
    const int64_t from = chunk + count * team / TEAMS, to = chunk + count * (team + 1) / TEAMS;
    float acc[EPV] = {};
    if (piece.in) {
#pragma unroll 8
        for (int64_t c = from; c < to; c++) {
            const uint64_t sums = (c == chunk ? a.tails : a.heads) + (uint64_t)(c * sums_stride(a.cols) + piece.at) * 4;
#pragma unroll
            for (int i = 0; i < EPV; i += 4) {
                const u32x4 v = *as_global<const u32x4_a4>(sums + i * 4);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i + j] += as_f(v[j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < EPV; i++) add[team][lane][i] = acc[i];
    __syncthreads();
    if (team > 0) return;
#pragma unroll 4
    for (int t = 1; t < TEAMS; t++)
#pragma unroll
        for (int i = 0; i < EPV; i++) acc[i] += add[t][lane][i];
#pragma unroll
    for (int i = 0; i < EPV; i++) acc[i] *= a.scale;
    store_row<ESZ, NARROW, false>(a.dtable + (uint64_t)key * (uint64_t)a.cols * ESZ, piece, a.cols, Elem<T>::pack(acc));
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static bool narrow_row(int64_t cols, int size) { return cols * size < 16; }

// Lanes and vectors of a row that is looked up in one go; longer ones take several.  No more lanes than vectors: 300000 rows
// of 16 take 14.0 us with 8 lanes of two, 42 with 64; 65536 of 32 7.4 with 16 of two, 10.1 with 64; a token's row of 512 2.9.
static RowShape embedding_shape(int64_t vectors)
{
    if (vectors <= 8) return {8, 1};
    if (vectors <= 16) return {8, 2};
    if (vectors <= 32) return {16, 2};
    if (vectors <= 64) return {32, 2};
    if (vectors <= 256) return {64, 4};
    return {256, 2};
}
template <class T>
static const void *embedding_kernel(int64_t cols, RowShape shape)
{
    if (narrow_row(cols, Elem<T>::ESZ)) return (const void *)k_embedding<T, 8, 1, true>;
    return shape.team == 8    ? shape.nv == 1 ? (const void *)k_embedding<T, 8, 1, false> : (const void *)k_embedding<T, 8, 2, false>
           : shape.team == 16 ? (const void *)k_embedding<T, 16, 2, false>
           : shape.team == 32 ? (const void *)k_embedding<T, 32, 2, false>
           : shape.team == 64 ? (const void *)k_embedding<T, 64, 4, false>
                              : (const void *)k_embedding<T, 256, 2, false>;
}

// Lanes to a row of a chunk.
static int backward_team(int64_t vectors) { return vectors <= 8 ? 8 : vectors <= 16 ? 16 : vectors <= 32 ? 32 : 64; }
template <class T, int TEAM, bool NARROW>
static const void *backward_kernel(int chunk)
{
    return chunk == 16   ? (const void *)k_embedding_backward<T, TEAM, 16, NARROW>
           : chunk == 64 ? (const void *)k_embedding_backward<T, TEAM, 64, NARROW>
                         : (const void *)k_embedding_backward<T, TEAM, 256, NARROW>;
}
template <class T>
static const void *backward_kernel(int64_t cols, int team, int chunk)
{
    if (narrow_row(cols, Elem<T>::ESZ)) return backward_kernel<T, 8, true>(chunk);
    return team == 8    ? backward_kernel<T, 8, false>(chunk)
           : team == 16 ? backward_kernel<T, 16, false>(chunk)
           : team == 32 ? backward_kernel<T, 32, false>(chunk)
                        : backward_kernel<T, 64, false>(chunk);
}
template <class T>
static const void *join_kernel(int64_t cols, int team)
{
    if (narrow_row(cols, Elem<T>::ESZ)) return (const void *)k_embedding_join<T, 8, true>;
    return team == 8    ? (const void *)k_embedding_join<T, 8, false>
           : team == 16 ? (const void *)k_embedding_join<T, 16, false>
           : team == 32 ? (const void *)k_embedding_join<T, 32, false>
                        : (const void *)k_embedding_join<T, 64, false>;
}

extern "C" int tftq_embedding(int dtype, int id_bytes, const void *ids, int64_t n, const void *table, int64_t vocab, int64_t cols,
                              int64_t row_stride, float scale, void *out, int device, void *stream)
{
    if (!dtype_ok(dtype)) return TFTQ_E_DTYPE;
    if (!rows_ok(n, cols) || !rows_ok(vocab, 0)) return TFTQ_E_SHAPE;
    if (id_bytes != 4 && id_bytes != 8) return TFTQ_E_ARG;
    if (n == 0 || cols == 0) return 0;
    if (!ids || (vocab && !table) || !out || row_stride < (vocab > 1 ? cols : 0)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const int size = dtype_size(dtype);
    const RowShape shape = embedding_shape((cols * size + 15) / 16);
    const int teams = 256 / shape.team;
    EmbeddingArgs a = {(uint64_t)ids, (uint64_t)table, (uint64_t)out, row_stride * size, 0, n, vocab, (int)cols, id_bytes == 8, scale};
    const void *k = dtype == TFTQ_F32   ? embedding_kernel<float>(cols, shape)
                    : dtype == TFTQ_F16 ? embedding_kernel<f16_tag>(cols, shape)
                                        : embedding_kernel<bf16_tag>(cols, shape);
    const int64_t at_once = ROWS_THREADS / shape.team;
    for (; a.row0 < n; a.row0 += at_once) {
        void *args[] = {(void *)&a};
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)((std::min(at_once, n - a.row0) + teams - 1) / teams)), dim3(256), args, 0, (hipStream_t)stream)) return rc;
    }
    return 0;
}

// Tokens of a chunk: few, where the machine is not full without (2^17 lanes are 8 wavefronts to a compute unit); more, where
// their sums cost more than they hasten (with 16 these are a quarter of dy's bytes or half).  The gradient in us with 16, 64 and 256:
// 65536 tokens of 64 bf16 37, 50, 110; 65536 of 256 56, 58, 106; 8192 of 4096 66, 66, 107; 300000 of 128 82, 70, 114; 131072 of
// 1024 144, 111, 119; 300000 of 1024 278, 197, 199; 2000000 of 128 349, 216, 200, and where all tokens are one 2737, 822, 326.
// Few tokens (up to 8192) have few sums to join, however long they are, and stay with 16 for twice the work: even numbers, 8192
// tokens of 4096 67.5 and 72, 4096 of 8192 166 and 172; 65536 of 512, where half of the numbers are in a hundredth of the table, 70 and 59.
static int embedding_chunk(int64_t n, int64_t vectors)
{
    return n * vectors < 1 << (n <= 8192 ? 23 : 22) ? 16 : n * vectors < 1 << 25 ? 64 : 256;
}

extern "C" int64_t tftq_embedding_backward_workspace(int dtype, int64_t n, int64_t vocab, int64_t cols)
{
    if (!dtype_ok(dtype)) return TFTQ_E_DTYPE;
    if (!rows_ok(n, cols) || !rows_ok(vocab, 0)) return TFTQ_E_SHAPE;
    const int64_t chunk = embedding_chunk(n, (cols * dtype_size(dtype) + 15) / 16), chunks = (n + chunk - 1) / chunk, numbers = (n * 8 + 15) & ~(int64_t)15;
    return sort_workspace(n, vocab) + numbers + chunks * sums_stride(cols) * 8;
}

extern "C" int tftq_embedding_backward(int dtype, int id_bytes, const void *ids, int64_t n, int64_t skip, const void *dy, int64_t vocab,
                                       int64_t cols, float scale, void *dtable, void *workspace, int64_t workspace_bytes, int device, void *stream)
{
    const int64_t bytes = tftq_embedding_backward_workspace(dtype, n, vocab, cols);
    if (bytes < 0) return (int)bytes;
    if (id_bytes != 4 && id_bytes != 8) return TFTQ_E_ARG;
    if (vocab == 0 || cols == 0) return 0;
    if ((n && (!ids || !dy || !workspace || ((uintptr_t)workspace & 15))) || !dtable) return TFTQ_E_ARG;
    if (workspace_bytes < bytes) return TFTQ_E_SIZE;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    hipStream_t st = (hipStream_t)stream;
    const int size = dtype_size(dtype);
    const int64_t vectors = (cols * size + 15) / 16;
    const int team = backward_team(vectors), teams = 256 / team;
    const int64_t across = (vectors + team - 1) / team;
    const uint64_t keys = (uint64_t)workspace + (uint64_t)sort_workspace(n, vocab), order = keys + (uint64_t)n * 4;
    TableArgs a = {};
    a.dy = (uint64_t)dy;
    a.keys = keys;
    a.order = order;
    a.dtable = (uint64_t)dtable;
    a.n = n;
    a.chunk = embedding_chunk(n, vectors);
    a.chunks = (n + a.chunk - 1) / a.chunk;
    a.heads = (keys + (uint64_t)n * 8 + 15) & ~(uint64_t)15;
    a.tails = a.heads + (uint64_t)(a.chunks * sums_stride(cols)) * 4;
    a.vocab = vocab;
    a.cols = (int)cols;
    a.across = (int)across;
    a.scale = scale;
    const SortArgs sort = {(uint64_t)ids, id_bytes == 8, n, (u32)vocab, skip >= 0 && skip < vocab ? (u32)skip : (u32)vocab, keys, order, 0, 0,
                           (uint64_t)dtable, vocab * cols * size};
    if (const int rc = sort_numbers(sort, workspace, st)) return rc;
    if (n == 0) return 0;
    auto launch = [&](const void *k, int64_t groups) {  // of all columns each
        const int64_t at_once = ROWS_THREADS / 256 / across;
        void *args[] = {(void *)&a};
        for (a.first = 0; a.first < groups; a.first += at_once)
            if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)(std::min(at_once, groups - a.first) * across)), dim3(256), args, 0, st)) return rc;
        return 0;
    };
    const void *k = dtype == TFTQ_F32   ? backward_kernel<float>(cols, team, a.chunk)
                    : dtype == TFTQ_F16 ? backward_kernel<f16_tag>(cols, team, a.chunk)
                                        : backward_kernel<bf16_tag>(cols, team, a.chunk);
    if (const int rc = launch(k, (a.chunks + teams - 1) / teams)) return rc;
    if (a.chunks < 2) return 0;
    k = dtype == TFTQ_F32 ? join_kernel<float>(cols, team) : dtype == TFTQ_F16 ? join_kernel<f16_tag>(cols, team) : join_kernel<bf16_tag>(cols, team);
    return launch(k, a.chunks - 1);
}
