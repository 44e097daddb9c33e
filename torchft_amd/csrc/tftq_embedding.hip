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
// chunk, and leaves fp32 sums where it goes on outside (at most one of each end).  A second launch goes over
// the table: rows of no token are filled with zeros, rows of several chunks add up their sums.  Every row is
// written once, whatever was there.
#include "tftq_sort.h"

struct EmbeddingArgs {
    uint64_t ids, table, out;
    int64_t stride;  // bytes from row to row of the table
    int64_t row0, rows;
    int64_t vocab;
    int cols, wide;
    float scale;
};

template <class T, int TEAM>
__global__ __launch_bounds__(256) void k_embedding(const EmbeddingArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, U = 4;
    const int lane = threadIdx.x % TEAM;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (row >= a.rows) return;
    const int64_t id = a.wide ? as_global<const int64_t>(a.ids)[row] : as_global<const int32_t>(a.ids)[row];
    const bool inside = id >= 0 && id < a.vocab;
    const uint64_t from = a.table + (uint64_t)(id * a.stride), to = a.out + (uint64_t)(row * a.cols) * ESZ;
    for (int col = lane * EPV; col < a.cols; col += U * TEAM * EPV) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = inside ? load_row<ESZ, false>(from, col + u * TEAM * EPV, a.cols) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < U; u++) {
            float f[EPV];
            Elem<T>::unpack(raw[u], f);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] *= a.scale;
            store_row<ESZ>(to, col + u * TEAM * EPV, a.cols, Elem<T>::pack(f));
        }
    }
}

struct TableArgs {
    uint64_t dy, keys, order, heads, tails, dtable;  // heads, tails: fp32 [chunks][cols]
    int64_t n, chunks, chunk0, vocab, row0;
    int cols, chunk, rows, across;  // tokens of a chunk, rows of the table for a workgroup, teams across the columns
    float scale;
};

// A lane sums the columns of one vector over a chunk; neighbouring workgroups are `across` parts of the same chunks.
template <class T, int TEAM>
__global__ __launch_bounds__(256) void k_embedding_chunks(const TableArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, U = 8;
    int64_t chunk = a.chunk0 + (int64_t)(blockIdx.x / (u32)a.across) * TEAMS + (TEAM < 256 ? threadIdx.x / TEAM : 0);
    if (TEAM == 64) chunk = __builtin_amdgcn_readfirstlane((int)chunk);  // a wavefront's: keys and places in scalar registers
    if (chunk >= a.chunks) return;
    const int col = (int)(blockIdx.x % (u32)a.across * TEAM + threadIdx.x % TEAM) * EPV;
    if (col >= a.cols) return;
    const GLOBAL u32 *keys = as_global<const u32>(a.keys), *order = as_global<const u32>(a.order);
    const int64_t begin = chunk * a.chunk, end = begin + a.chunk < a.n ? begin + a.chunk : a.n;
    const u32 none = 0xFFFFFFFFu;
    const u32 previous = begin > 0 ? keys[begin - 1] : none, next = end < a.n ? keys[end] : none;
    float acc[EPV] = {};
    u32 current = none;

    auto leave = [&](bool last) {  // the run of `current` ends, or the chunk does
        if (current == none || current >= (u32)a.vocab) return;
        const bool goes_on = last && next == current;
        if (current != previous && !goes_on) {
            float f[EPV];
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] = acc[i] * a.scale;
            store_row<ESZ>(a.dtable + (uint64_t)current * (uint64_t)a.cols * ESZ, col, a.cols, Elem<T>::pack(f));
            return;
        }
        const uint64_t sums = (current == previous ? a.heads : a.tails) + (uint64_t)(chunk * a.cols) * 4;
#pragma unroll
        for (int i = 0; i < EPV; i += 4)
            store_row<4, false>(sums, col + i, a.cols, u32x4{as_u(acc[i]), as_u(acc[i + 1]), as_u(acc[i + 2]), as_u(acc[i + 3])});
    };
    for (int64_t at = begin; at < end; at += U) {
        u32x4 raw[U];
        u32 key[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            key[u] = at + u < end ? keys[at + u] : none;
            raw[u] = u32x4{0, 0, 0, 0};
            if (key[u] < (u32)a.vocab) raw[u] = load_row<ESZ>(a.dy + (uint64_t)order[at + u] * (uint64_t)a.cols * ESZ, col, a.cols);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (key[u] == none) continue;
            if (key[u] != current) {
                leave(false);
                current = key[u];
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

// The table's rows: zeros where no token is, the chunks' sums where there are several.
template <class T, int TEAM>
__global__ __launch_bounds__(256) void k_embedding_table(const TableArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM;
    __shared__ int64_t starts[256];
    const int64_t first = a.row0 + (int64_t)blockIdx.x * a.rows;
    if ((int)threadIdx.x <= a.rows) starts[threadIdx.x] = first_at(as_global<const u32>(a.keys), a.n, first + threadIdx.x);
    __syncthreads();
    const int lane = threadIdx.x % TEAM;
    for (int r = threadIdx.x / TEAM; r < a.rows && first + r < a.vocab; r += TEAMS) {
        const int64_t s = starts[r], e = starts[r + 1];
        const uint64_t to = a.dtable + (uint64_t)(first + r) * (uint64_t)a.cols * ESZ;
        if (s == e) {
            for (int col = lane * EPV; col < a.cols; col += TEAM * EPV) store_row<ESZ>(to, col, a.cols, u32x4{0, 0, 0, 0});
            continue;
        }
        const int64_t c0 = s / a.chunk, c1 = (e - 1) / a.chunk;
        if (c0 == c1) continue;  // written with its chunk
        for (int col = lane * EPV; col < a.cols; col += TEAM * EPV) {
            float acc[EPV];
#pragma unroll
            for (int i = 0; i < EPV; i++) acc[i] = 0.0f;
#pragma unroll 4
            for (int64_t c = c0; c <= c1; c++) {
                const uint64_t sums = (c == c0 ? a.tails : a.heads) + (uint64_t)(c * a.cols) * 4;
#pragma unroll
                for (int i = 0; i < EPV; i += 4) {
                    const u32x4 v = load_row<4, false>(sums, col + i, a.cols);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i + j] += as_f(v[j]);
                }
            }
#pragma unroll
            for (int i = 0; i < EPV; i++) acc[i] *= a.scale;
            store_row<ESZ>(to, col, a.cols, Elem<T>::pack(acc));
        }
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static int embedding_team(int64_t vectors) { return vectors <= 8 ? 8 : vectors <= 64 ? 64 : 256; }

#define EMBEDDING_KERNEL(K, dtype, team)                                                                                  \
    (dtype == TFTQ_F32   ? team == 8 ? (const void *)K<float, 8> : team == 64 ? (const void *)K<float, 64> : (const void *)K<float, 256>            \
     : dtype == TFTQ_F16 ? team == 8 ? (const void *)K<f16_tag, 8> : team == 64 ? (const void *)K<f16_tag, 64> : (const void *)K<f16_tag, 256>      \
                         : team == 8 ? (const void *)K<bf16_tag, 8> : team == 64 ? (const void *)K<bf16_tag, 64> : (const void *)K<bf16_tag, 256>)

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
    const int size = dtype_size(dtype), team = embedding_team((cols * size + 15) / 16), teams = 256 / team;
    EmbeddingArgs a = {(uint64_t)ids, (uint64_t)table, (uint64_t)out, row_stride * size, 0, n, vocab, (int)cols, id_bytes == 8, scale};
    const void *k = EMBEDDING_KERNEL(k_embedding, dtype, team);
    const int64_t at_once = ROWS_THREADS / team;
    for (; a.row0 < n; a.row0 += at_once) {
        void *args[] = {(void *)&a};
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)((std::min(at_once, n - a.row0) + teams - 1) / teams)), dim3(256), args, 0, (hipStream_t)stream)) return rc;
    }
    return 0;
}

// Tokens of a chunk: 32, and with more than 8192 tokens as many as there are chunks for every eight, so that neither a
// chunk nor the sums of one row are long.
static int embedding_chunk(int64_t n)
{
    int chunk = 32;
    while ((int64_t)chunk * chunk * 8 < n) chunk *= 2;
    return chunk;
}

extern "C" int64_t tftq_embedding_backward_workspace(int64_t n, int64_t vocab, int64_t cols)
{
    if (!rows_ok(n, cols) || !rows_ok(vocab, 0)) return TFTQ_E_SHAPE;
    const int64_t chunks = (n + embedding_chunk(n) - 1) / embedding_chunk(n), numbers = (n * 8 + 15) & ~(int64_t)15;
    return sort_workspace(n, vocab) + numbers + chunks * cols * 8;
}

extern "C" int tftq_embedding_backward(int dtype, int id_bytes, const void *ids, int64_t n, int64_t skip, const void *dy, int64_t vocab,
                                       int64_t cols, float scale, void *dtable, void *workspace, int64_t workspace_bytes, int device, void *stream)
{
    if (!dtype_ok(dtype)) return TFTQ_E_DTYPE;
    const int64_t bytes = tftq_embedding_backward_workspace(n, vocab, cols);
    if (bytes < 0) return (int)bytes;
    if (id_bytes != 4 && id_bytes != 8) return TFTQ_E_ARG;
    if (vocab == 0 || cols == 0) return 0;
    if ((n && (!ids || !dy || !workspace || ((uintptr_t)workspace & 15))) || !dtable) return TFTQ_E_ARG;
    if (workspace_bytes < bytes) return TFTQ_E_SIZE;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    hipStream_t st = (hipStream_t)stream;
    const int size = dtype_size(dtype), team = embedding_team((cols * size + 15) / 16), teams = 256 / team;
    const int64_t vectors = (cols * size + 15) / 16, across = (vectors + team - 1) / team;
    const uint64_t keys = (uint64_t)workspace + (uint64_t)sort_workspace(n, vocab), order = keys + (uint64_t)n * 4;
    TableArgs a = {};
    a.dy = (uint64_t)dy;
    a.keys = keys;
    a.order = order;
    a.dtable = (uint64_t)dtable;
    a.n = n;
    a.chunk = embedding_chunk(n);
    a.chunks = (n + a.chunk - 1) / a.chunk;
    a.heads = (keys + (uint64_t)n * 8 + 15) & ~(uint64_t)15;
    a.tails = a.heads + (uint64_t)(a.chunks * cols) * 4;
    a.vocab = vocab;
    a.cols = (int)cols;
    a.across = (int)across;
    a.scale = scale;
    void *args[] = {(void *)&a};
    if (n) {
        const SortArgs s = {(uint64_t)ids, id_bytes == 8, n, (u32)vocab, skip >= 0 && skip < vocab ? (u32)skip : (u32)vocab, keys, order, 0, 0};
        if (const int rc = sort_numbers(s, workspace, st)) return rc;
        const void *k = EMBEDDING_KERNEL(k_embedding_chunks, dtype, team);
        const int64_t at_once = std::max<int64_t>(1, ROWS_THREADS / 256 / across) * teams;
        for (; a.chunk0 < a.chunks; a.chunk0 += at_once)
            if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)((std::min(at_once, a.chunks - a.chunk0) + teams - 1) / teams * across)),
                                                    dim3(256), args, 0, st))
                return rc;
    }
    // 64 KB of the table to a workgroup, 255 rows at most: the search for where its rows' tokens begin is one for all
    const int64_t row_bytes = cols * size;
    a.rows = (int)std::min<int64_t>(255, std::max<int64_t>(teams, 65536 / row_bytes));
    const void *k = EMBEDDING_KERNEL(k_embedding_table, dtype, team);
    const int64_t groups = (vocab + a.rows - 1) / a.rows, at_once = ROWS_THREADS / 256;
    for (int64_t done = 0; done < groups; done += at_once) {
        a.row0 = done * a.rows;
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)std::min(at_once, groups - done)), dim3(256), args, 0, st)) return rc;
    }
    return 0;
}
