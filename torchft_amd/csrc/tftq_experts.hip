// Tokens to experts and back: choices sorted by expert, the tokens' rows there, and the experts' rows back with
// weights, with the gradients of both.
//
// Token t makes choices (t, 0) to (t, k - 1); a stable counting sort (tftq_sort.h) gives every choice its place, so that
// an expert's choices lie side by side in the order of their tokens.  A choice that names no expert has its place
// behind all others.
//
//    dispatch   out[place(t, s)] = x[t]                          zeros in places without an expert
//    combine    y[t] = sum over s of w[t, s] rows[place(t, s)]   (choices without an expert left out)
//    backward   drows[place(t, s)] = w[t, s] dy[t];  dw[t, s] = <dy[t], rows[place(t, s)]>
//
// The gradient of dispatch is combine without weights.  All go token by token, not place by place: a token's row is read
// once for all its choices, sums over the choices are one lane's, in their order, and need no atomics.  They are
// bound by memory; rows of the k places are whole lines wherever they lie.
#include "tftq_sort.h"

struct ExpertArgs {
    uint64_t x, rows, weights, position, used, y, drows, dweights;  // weights: 0 for ones.  used: where the count of places with an expert is
    int64_t x_stride;                                               // bytes from row to row of x, of rows and of dy
    int64_t rows_stride;
    int64_t token0, tokens;
    int cols, k, wide;  // wide: the weights are fp32 and the rows are not
};

// How many places have an expert: whatever memory says, no more than there are.
DEV u32 places_used(const ExpertArgs &a) { return min(*as_global<const u32>(a.used), (u32)(a.tokens * a.k)); }

// x [tokens] -> y [tokens k] by places; elements of ESZ bytes.  8192x4096 bf16 to two of eight 33.7 us, 202 MB, 6.0 TB/s (stores that
// stream past the caches, at scattered places, 37.7); 4099x777 fp32 to six of 61 15.8, 5.7.
template <int ESZ, int TEAM, int U, bool NARROW>
__global__ __launch_bounds__(256) void k_dispatch(const ExpertArgs a)
{
    constexpr int EPV = 16 / ESZ, TEAMS = 256 / TEAM;
    const int lane = threadIdx.x % TEAM;
    const int64_t token = a.token0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (token >= a.tokens) return;
    const u32 used = places_used(a);
    const GLOBAL u32 *position = as_global<const u32>(a.position) + token * a.k;
    const uint64_t from = a.x + (uint64_t)(token * a.x_stride);
    for (int col = lane * EPV; col < a.cols; col += U * TEAM * EPV) {
        Piece p[U];
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            p[u] = piece_of<EPV, NARROW>(col + u * TEAM * EPV, a.cols);
            raw[u] = load_row<ESZ, NARROW>(from, p[u], a.cols);
        }
        for (int s = 0; s < a.k; s++) {
            const u32 place = position[s];
            if (place >= (u32)(a.tokens * a.k)) continue;
            const uint64_t to = a.y + (uint64_t)place * (uint64_t)a.cols * ESZ;
#pragma unroll
            for (int u = 0; u < U; u++) store_row<ESZ, NARROW, false>(to, p[u], a.cols, place < used ? raw[u] : u32x4{0, 0, 0, 0});
        }
    }
}

template <class T>
DEV float expert_weight(const ExpertArgs &a, int64_t choice)
{
    if (!a.weights) return 1.0f;
    return a.wide ? as_global<const float>(a.weights)[choice] : Elem<T>::load(a.weights, choice);
}

// Four choices at a time are on their way.  8192x4096 bf16 from two 34.1 us, 202 MB, 5.9 TB/s; 4099x777 fp32 from six 17.3, 5.1.
template <class T, int TEAM, int U, bool NARROW>
__global__ __launch_bounds__(256) void k_combine(const ExpertArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, S = 4;
    const int lane = threadIdx.x % TEAM;
    const int64_t token = a.token0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (token >= a.tokens) return;
    const u32 used = places_used(a);
    const int64_t choice = token * a.k;
    const uint64_t to = a.y + (uint64_t)(token * a.cols) * ESZ;
    for (int col = lane * EPV; col < a.cols; col += U * TEAM * EPV) {
        float acc[U][EPV] = {};
        for (int s0 = 0; s0 < a.k; s0 += S) {
            u32 place[S];
            float w[S];
            u32x4 raw[S][U];
#pragma unroll
            for (int s = 0; s < S; s++) {
                const bool there = s0 + s < a.k;
                place[s] = there ? as_global<const u32>(a.position)[choice + s0 + s] : used;
                w[s] = there ? expert_weight<T>(a, choice + s0 + s) : 0.0f;
            }
#pragma unroll
            for (int s = 0; s < S; s++) {
                // of a choice without an expert nothing is read, and its weight leaves it at nothing
                const bool live = place[s] < used;
                if (!live) w[s] = 0.0f;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    Piece p = piece_of<EPV, NARROW>(col + u * TEAM * EPV, a.cols);
                    p.in = p.in && live;
                    raw[s][u] = load_row<ESZ, NARROW>(a.rows + (uint64_t)place[s] * (uint64_t)a.rows_stride, p, a.cols);
                }
            }
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float f[EPV];
                    Elem<T>::unpack(raw[s][u], f);
#pragma unroll
                    for (int i = 0; i < EPV; i++) acc[u][i] = __builtin_fmaf(w[s], f[i], acc[u][i]);
                }
        }
#pragma unroll
        for (int u = 0; u < U; u++) store_row<ESZ, NARROW>(to, piece_of<EPV, NARROW>(col + u * TEAM * EPV, a.cols), a.cols, Elem<T>::pack(acc[u]));
    }
}

// x is dy.  NV: vectors of dy that a lane keeps for all choices, and of the rows of two choices that are on their way; MORE:
// the row is longer, and read again for every choice.  8192x4096 bf16 56 us, 336 MB, 6.0 TB/s; 4099x777 fp32 and six 35.4, 4.7.
template <class T, int TEAM, int NV, bool NARROW, bool MORE>
__global__ __launch_bounds__(256) void k_combine_backward(const ExpertArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, S = 2;
    __shared__ float lds[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    const int lane = threadIdx.x % TEAM;
    const int64_t token = a.token0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (token >= a.tokens) return;
    const u32 used = places_used(a);
    const uint64_t from = a.x + (uint64_t)(token * a.x_stride);
    Piece piece[NV];
    u32x4 dy[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        piece[v] = piece_of<EPV, NARROW>((v * TEAM + lane) * EPV, a.cols);
        dy[v] = load_row<ESZ, NARROW, !MORE>(from, piece[v], a.cols);
    }
    for (int s0 = 0; s0 < a.k; s0 += S) {
        u32 place[S];
        float w[S], dot[S];
        bool live[S];
#pragma unroll
        for (int s = 0; s < S; s++) {
            const int64_t choice = token * a.k + s0 + s;
            const bool there = s0 + s < a.k;
            place[s] = there ? as_global<const u32>(a.position)[choice] : used;
            live[s] = place[s] < used;
            w[s] = live[s] ? expert_weight<T>(a, choice) : 0.0f;
            dot[s] = 0.0f;
        }
        for (int base = 0; base < (MORE ? a.cols : 1); base += NV * TEAM * EPV) {
            if (MORE && (base > 0 || s0 > 0)) {
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    piece[v] = piece_of<EPV, NARROW>(base + (v * TEAM + lane) * EPV, a.cols);
                    dy[v] = load_row<ESZ, NARROW, false>(from, piece[v], a.cols);
                }
            }
            u32x4 raw[S][NV];
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    Piece p = piece[v];
                    p.in = p.in && live[s] && a.dweights;
                    raw[s][v] = load_row<ESZ, NARROW>(a.rows + (uint64_t)place[s] * (uint64_t)a.rows_stride, p, a.cols);
                }
#pragma unroll
            for (int v = 0; v < NV; v++) {
                float d[EPV], once[EPV];
                Elem<T>::unpack(dy[v], d);
                Elem<T>::unpack(dy[v], once);
                if (!NARROW) count_once(once, piece[v]);
#pragma unroll
                for (int s = 0; s < S; s++) {
                    if (s0 + s >= a.k) continue;
                    float f[EPV], out[EPV];
                    Elem<T>::unpack(raw[s][v], f);
                    if (!NARROW) count_once(f, piece[v]);  // no 0 times infinity
#pragma unroll
                    for (int i = 0; i < EPV; i++) {
                        dot[s] = __builtin_fmaf(once[i], f[i], dot[s]);
                        out[i] = live[s] ? d[i] * w[s] : 0.0f;
                    }
                    Piece p = piece[v];
                    p.in = p.in && place[s] < (u32)(a.tokens * a.k);  // a branch over all of this instead: 8 % slower
                    if (a.drows) store_row<ESZ, NARROW, false>(a.drows + (uint64_t)place[s] * (uint64_t)a.cols * ESZ, p, a.cols, Elem<T>::pack(out));
                }
            }
        }
        if (!a.dweights) continue;
        team_sum2<TEAM>(dot[0], dot[1], lds);
        if (lane < S && s0 + lane < a.k) {
            const int64_t choice = token * a.k + s0 + lane;
            const bool taken = lane ? live[1] : live[0];
            const float dw = taken ? lane ? dot[1] : dot[0] : 0.0f;
            if (a.wide) as_global<float>(a.dweights)[choice] = dw;
            else Elem<T>::store(a.dweights, choice, dw);
        }
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static bool experts_ok(int64_t tokens, int64_t k, int64_t cols)
{
    return rows_ok(tokens, cols) && k >= 0 && k <= ROWS_MOST && (k == 0 || tokens <= ROWS_MOST / k);
}
// Lanes and vectors of a row that is taken in one go; longer ones take several.  Four vectors a lane, unless they are fewer:
// 24594 rows of 195 (fp32) there 17 us with 64 lanes of four, 24 with 256; 262144 rows of 8 (bf16) back 7.2 with 8 lanes of
// one, 12.9 with four of each.
static RowShape expert_shape(int64_t vectors)
{
    if (vectors <= 8) return {8, 1};
    if (vectors <= 16) return {8, 2};
    if (vectors <= 32) return {8, 4};
    if (vectors <= 64) return {16, 4};
    if (vectors <= 128) return {64, 2};
    if (vectors <= 256) return {64, 4};
    return {256, 2};
}
#define EXPERT_SHAPES(K, X, size)                                        \
    (cols * size < 16    ? (const void *)K<X, 8, 1, true>                    \
     : shape.team == 8   ? shape.nv == 1   ? (const void *)K<X, 8, 1, false> \
                           : shape.nv == 2 ? (const void *)K<X, 8, 2, false> \
                                           : (const void *)K<X, 8, 4, false> \
     : shape.team == 16  ? (const void *)K<X, 16, 4, false>                  \
     : shape.team == 256 ? (const void *)K<X, 256, 2, false>                 \
     : shape.nv == 2     ? (const void *)K<X, 64, 2, false>                  \
                         : (const void *)K<X, 64, 4, false>)

static int expert_launch(const void *kernel, ExpertArgs a, int team, hipStream_t st)
{
    const int teams = 256 / team;
    const int64_t at_once = ROWS_THREADS / team;
    for (; a.token0 < a.tokens; a.token0 += at_once) {
        void *args[] = {(void *)&a};
        const int64_t now = std::min(at_once, a.tokens - a.token0);
        if (const int rc = (int)hipLaunchKernel(kernel, dim3((unsigned)((now + teams - 1) / teams)), dim3(256), args, 0, st)) return rc;
    }
    return 0;
}

extern "C" int64_t tftq_expert_sort_workspace(int64_t choices, int64_t experts)
{
    if (!rows_ok(choices, experts)) return TFTQ_E_SHAPE;
    return sort_workspace(choices, experts) + (sort_needs_keys(choices, experts) ? (choices * 4 + 15) & ~(int64_t)15 : 0);
}

extern "C" int tftq_expert_sort(int id_bytes, const void *chosen, int64_t choices, int64_t experts, int32_t *order, int32_t *position,
                                int32_t *offsets, void *workspace, int64_t workspace_bytes, int device, void *stream)
{
    const int64_t bytes = tftq_expert_sort_workspace(choices, experts);
    if (bytes < 0) return (int)bytes;
    if (id_bytes != 4 && id_bytes != 8) return TFTQ_E_ARG;
    if (!offsets || (choices && (!chosen || !order || !position)) || (bytes && (!workspace || ((uintptr_t)workspace & 15)))) return TFTQ_E_ARG;
    if (workspace_bytes < bytes) return TFTQ_E_SIZE;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const SortArgs a = {(uint64_t)chosen, id_bytes == 8, choices, (u32)experts, (u32)experts,
                        sort_needs_keys(choices, experts) ? (uint64_t)workspace + (uint64_t)sort_workspace(choices, experts) : 0, (uint64_t)order, (uint64_t)position, (uint64_t)offsets, 0, 0};
    return sort_numbers(a, workspace, (hipStream_t)stream);
}

extern "C" int tftq_dispatch(int element_bytes, const void *x, int64_t x_stride, int64_t tokens, int64_t k, int64_t cols, const int32_t *position,
                             const int32_t *used, void *out, int device, void *stream)
{
    if (element_bytes != 1 && element_bytes != 2 && element_bytes != 4) return TFTQ_E_DTYPE;
    if (!experts_ok(tokens, k, cols)) return TFTQ_E_SHAPE;
    if (tokens == 0 || k == 0 || cols == 0) return 0;
    if (!x || !position || !used || !out || x_stride < (tokens > 1 ? cols : 0)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const RowShape shape = expert_shape((cols * element_bytes + 15) / 16);
    ExpertArgs a = {};
    a.x = (uint64_t)x;
    a.x_stride = x_stride * element_bytes;
    a.position = (uint64_t)position;
    a.used = (uint64_t)used;
    a.y = (uint64_t)out;
    a.tokens = tokens;
    a.cols = (int)cols;
    a.k = (int)k;
#define K(ESZ) EXPERT_SHAPES(k_dispatch, ESZ, ESZ)
    return expert_launch(element_bytes == 1 ? K(1) : element_bytes == 2 ? K(2) : K(4), a, shape.team, (hipStream_t)stream);
#undef K
}

extern "C" int tftq_combine(int dtype, int weight_dtype, const void *rows, int64_t rows_stride, const void *weights, int64_t tokens, int64_t k,
                            int64_t cols, const int32_t *position, const int32_t *used, void *out, int device, void *stream)
{
    if (!dtype_ok(dtype) || (weights && weight_dtype != dtype && weight_dtype != TFTQ_F32)) return TFTQ_E_DTYPE;
    if (!experts_ok(tokens, k, cols)) return TFTQ_E_SHAPE;
    if (tokens == 0 || cols == 0) return 0;
    if ((k && (!rows || !position)) || !used || !out || rows_stride < (tokens * k > 1 ? cols : 0)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const int size = dtype_size(dtype);
    const RowShape shape = expert_shape((cols * size + 15) / 16);
    ExpertArgs a = {};
    a.rows = (uint64_t)rows;
    a.rows_stride = rows_stride * size;
    a.weights = (uint64_t)weights;
    a.wide = weights && weight_dtype != dtype;
    a.position = (uint64_t)position;
    a.used = (uint64_t)used;
    a.y = (uint64_t)out;
    a.tokens = tokens;
    a.cols = (int)cols;
    a.k = (int)k;
#define K(T) EXPERT_SHAPES(k_combine, T, size)
    return expert_launch(dtype == TFTQ_F32 ? K(float) : dtype == TFTQ_F16 ? K(f16_tag) : K(bf16_tag), a, shape.team, (hipStream_t)stream);
#undef K
}

extern "C" int tftq_combine_backward(int dtype, int weight_dtype, const void *dy, int64_t dy_stride, const void *rows, int64_t rows_stride,
                                     const void *weights, int64_t tokens, int64_t k, int64_t cols, const int32_t *position, const int32_t *used,
                                     void *drows, void *dweights, int device, void *stream)
{
    if (!dtype_ok(dtype) || (weights && weight_dtype != dtype && weight_dtype != TFTQ_F32)) return TFTQ_E_DTYPE;
    if (!experts_ok(tokens, k, cols)) return TFTQ_E_SHAPE;
    if (tokens == 0 || k == 0 || (cols == 0 && !dweights)) return 0;
    if ((cols && (!dy || (dweights && !rows))) || !position || !used || (!drows && !dweights) || (dweights && !weights)) return TFTQ_E_ARG;
    if (dy_stride < (tokens > 1 ? cols : 0) || (dweights && rows_stride < (tokens * k > 1 ? cols : 0))) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const int size = dtype_size(dtype);
    const int64_t vectors = (cols * size + 15) / 16;
    const RowShape shape = expert_shape(vectors);
    const int per_lane = (int)std::min<int64_t>(5, (vectors + shape.team - 1) / shape.team);
    ExpertArgs a = {};
    a.x = (uint64_t)dy;
    a.x_stride = dy_stride * size;
    a.rows = (uint64_t)rows;
    a.rows_stride = rows_stride * size;
    a.weights = (uint64_t)weights;
    a.wide = weights && weight_dtype != dtype;
    a.position = (uint64_t)position;
    a.used = (uint64_t)used;
    a.drows = (uint64_t)drows;
    a.dweights = (uint64_t)dweights;
    a.tokens = tokens;
    a.cols = (int)cols;
    a.k = (int)k;
#define K(T)                                                                                          \
    (cols * size < 16    ? (const void *)k_combine_backward<T, 8, 1, true, false>                         \
     : shape.team == 8   ? shape.nv == 1   ? (const void *)k_combine_backward<T, 8, 1, false, false>      \
                           : shape.nv == 2 ? (const void *)k_combine_backward<T, 8, 2, false, false>      \
                                           : (const void *)k_combine_backward<T, 8, 4, false, false>      \
     : shape.team == 16  ? (const void *)k_combine_backward<T, 16, 4, false, false>                       \
     : shape.team == 64  ? shape.nv == 2 ? (const void *)k_combine_backward<T, 64, 2, false, false>       \
                                         : (const void *)k_combine_backward<T, 64, 4, false, false>       \
     : per_lane <= 2     ? (const void *)k_combine_backward<T, 256, 2, false, false>                      \
     : per_lane <= 4     ? (const void *)k_combine_backward<T, 256, 4, false, false>                      \
                         : (const void *)k_combine_backward<T, 256, 4, false, true>)
    return expert_launch(dtype == TFTQ_F32 ? K(float) : dtype == TFTQ_F16 ? K(f16_tag) : K(bf16_tag), a, shape.team, (hipStream_t)stream);
#undef K
}
