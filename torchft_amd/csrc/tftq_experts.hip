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

// x [tokens] -> y [tokens k] by places; elements of ESZ bytes.
template <int ESZ, int TEAM>
__global__ __launch_bounds__(256) void k_dispatch(const ExpertArgs a)
{
    constexpr int EPV = 16 / ESZ, TEAMS = 256 / TEAM, U = 4;
    const int lane = threadIdx.x % TEAM;
    const int64_t token = a.token0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (token >= a.tokens) return;
    const u32 used = *as_global<const u32>(a.used);
    const GLOBAL u32 *position = as_global<const u32>(a.position) + token * a.k;
    const uint64_t from = a.x + (uint64_t)(token * a.x_stride);
    for (int col = lane * EPV; col < a.cols; col += U * TEAM * EPV) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = load_row<ESZ>(from, col + u * TEAM * EPV, a.cols);
        for (int s = 0; s < a.k; s++) {
            const u32 place = position[s];
            const uint64_t to = a.y + (uint64_t)place * (uint64_t)a.cols * ESZ;
#pragma unroll
            for (int u = 0; u < U; u++) store_row<ESZ>(to, col + u * TEAM * EPV, a.cols, place < used ? raw[u] : u32x4{0, 0, 0, 0});
        }
    }
}

template <class T>
DEV float expert_weight(const ExpertArgs &a, int64_t choice)
{
    if (!a.weights) return 1.0f;
    return a.wide ? as_global<const float>(a.weights)[choice] : Elem<T>::load(a.weights, choice);
}

template <class T, int TEAM>
__global__ __launch_bounds__(256) void k_combine(const ExpertArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, U = 2;
    const int lane = threadIdx.x % TEAM;
    const int64_t token = a.token0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (token >= a.tokens) return;
    const u32 used = *as_global<const u32>(a.used);
    const GLOBAL u32 *position = as_global<const u32>(a.position) + token * a.k;
    const uint64_t to = a.y + (uint64_t)(token * a.cols) * ESZ;
    for (int col = lane * EPV; col < a.cols; col += U * TEAM * EPV) {
        float acc[U][EPV] = {};
#pragma unroll 2
        for (int s = 0; s < a.k; s++) {
            const u32 place = position[s];
            if (place >= used) continue;
            const uint64_t from = a.rows + (uint64_t)place * (uint64_t)a.rows_stride;
            const float w = expert_weight<T>(a, token * a.k + s);
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = load_row<ESZ>(from, col + u * TEAM * EPV, a.cols);
#pragma unroll
            for (int u = 0; u < U; u++) {
                float f[EPV];
                Elem<T>::unpack(raw[u], f);
#pragma unroll
                for (int i = 0; i < EPV; i++) acc[u][i] = __builtin_fmaf(w, f[i], acc[u][i]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) store_row<ESZ>(to, col + u * TEAM * EPV, a.cols, Elem<T>::pack(acc[u]));
    }
}

// x is dy.  NV: vectors of dy that a lane keeps for all choices; 0: read again for every one.
template <class T, int TEAM, int NV>
__global__ __launch_bounds__(256) void k_combine_backward(const ExpertArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM;
    __shared__ float lds[TEAM > 64 ? TEAM / 64 : 1];
    const int lane = threadIdx.x % TEAM;
    const int64_t token = a.token0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (token >= a.tokens) return;
    const u32 used = *as_global<const u32>(a.used);
    const uint64_t from = a.x + (uint64_t)(token * a.x_stride);
    u32x4 dy[NV > 0 ? NV : 1];
#pragma unroll
    for (int v = 0; v < NV; v++) dy[v] = load_row<ESZ>(from, (v * TEAM + lane) * EPV, a.cols);
    for (int s = 0; s < a.k; s++) {
        const int64_t choice = token * a.k + s;
        const u32 place = as_global<const u32>(a.position)[choice];
        const bool live = place < used;
        const float w = live ? expert_weight<T>(a, choice) : 0.0f;
        const uint64_t row = a.rows + (uint64_t)place * (uint64_t)a.rows_stride, to = a.drows + (uint64_t)place * (uint64_t)a.cols * ESZ;
        float dot = 0.0f;
        auto step = [&](const u32x4 g, int col) {
            u32x4 r = {0, 0, 0, 0};
            if (live && a.dweights) r = load_row<ESZ>(row, col, a.cols);
            float f[EPV], d[EPV];
            Elem<T>::unpack(r, f);
            Elem<T>::unpack(g, d);
#pragma unroll
            for (int i = 0; i < EPV; i++) {
                dot = __builtin_fmaf(d[i], f[i], dot);
                d[i] = live ? d[i] * w : 0.0f;
            }
            if (a.drows) store_row<ESZ>(to, col, a.cols, Elem<T>::pack(d));
        };
        if (NV > 0) {
#pragma unroll
            for (int v = 0; v < NV; v++) step(dy[v], (v * TEAM + lane) * EPV);
        } else {
            for (int col = lane * EPV; col < a.cols; col += TEAM * EPV) step(load_row<ESZ, false>(from, col, a.cols), col);
        }
        if (!a.dweights) continue;
        dot = team_sum<TEAM>(dot, lds);
        if (lane == 0) {
            const float dw = live ? dot : 0.0f;
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
static int expert_team(int64_t vectors) { return vectors <= 8 ? 8 : vectors <= 128 ? 64 : 256; }

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
    return sort_workspace(choices, experts) + ((choices * 4 + 15) & ~(int64_t)15);
}

extern "C" int tftq_expert_sort(int id_bytes, const void *chosen, int64_t choices, int64_t experts, int32_t *order, int32_t *position,
                                int32_t *offsets, void *workspace, int64_t workspace_bytes, int device, void *stream)
{
    const int64_t bytes = tftq_expert_sort_workspace(choices, experts);
    if (bytes < 0) return (int)bytes;
    if (id_bytes != 4 && id_bytes != 8) return TFTQ_E_ARG;
    if (!offsets || (choices && (!chosen || !order || !position || !workspace || ((uintptr_t)workspace & 15)))) return TFTQ_E_ARG;
    if (workspace_bytes < bytes) return TFTQ_E_SIZE;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const SortArgs a = {(uint64_t)chosen, id_bytes == 8, choices, (u32)experts, (u32)experts,
                        choices ? (uint64_t)workspace + (uint64_t)sort_workspace(choices, experts) : 0, (uint64_t)order, (uint64_t)position, (uint64_t)offsets};
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
    const int team = expert_team((cols * element_bytes + 15) / 16);
    ExpertArgs a = {};
    a.x = (uint64_t)x;
    a.x_stride = x_stride * element_bytes;
    a.position = (uint64_t)position;
    a.used = (uint64_t)used;
    a.y = (uint64_t)out;
    a.tokens = tokens;
    a.cols = (int)cols;
    a.k = (int)k;
#define K(ESZ) (team == 8 ? (const void *)k_dispatch<ESZ, 8> : team == 64 ? (const void *)k_dispatch<ESZ, 64> : (const void *)k_dispatch<ESZ, 256>)
    return expert_launch(element_bytes == 1 ? K(1) : element_bytes == 2 ? K(2) : K(4), a, team, (hipStream_t)stream);
#undef K
}

extern "C" int tftq_combine(int dtype, int weight_dtype, const void *rows, int64_t rows_stride, const void *weights, int64_t tokens, int64_t k,
                            int64_t cols, const int32_t *position, const int32_t *used, void *out, int device, void *stream)
{
    if (!dtype_ok(dtype) || (weights && weight_dtype != dtype && weight_dtype != TFTQ_F32)) return TFTQ_E_DTYPE;
    if (!experts_ok(tokens, k, cols)) return TFTQ_E_SHAPE;
    if (tokens == 0 || cols == 0) return 0;
    if ((k && (!rows || !position || !used)) || !out || rows_stride < (tokens * k > 1 ? cols : 0)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const int size = dtype_size(dtype), team = expert_team((cols * size + 15) / 16);
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
#define K(T) (team == 8 ? (const void *)k_combine<T, 8> : team == 64 ? (const void *)k_combine<T, 64> : (const void *)k_combine<T, 256>)
    return expert_launch(dtype == TFTQ_F32 ? K(float) : dtype == TFTQ_F16 ? K(f16_tag) : K(bf16_tag), a, team, (hipStream_t)stream);
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
    const int team = expert_team(vectors), nv = vectors <= team ? 1 : vectors <= 2 * team ? 2 : vectors <= 4 * team ? 4 : 0;
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
#define K(T)                                                                                                          \
    (team == 8    ? (const void *)k_combine_backward<T, 8, 1>                                                         \
     : team == 64 ? nv == 1 ? (const void *)k_combine_backward<T, 64, 1> : (const void *)k_combine_backward<T, 64, 2> \
     : nv == 1    ? (const void *)k_combine_backward<T, 256, 1>                                                       \
     : nv == 2    ? (const void *)k_combine_backward<T, 256, 2>                                                       \
     : nv == 4    ? (const void *)k_combine_backward<T, 256, 4>                                                       \
                  : (const void *)k_combine_backward<T, 256, 0>)
    return expert_launch(dtype == TFTQ_F32 ? K(float) : dtype == TFTQ_F16 ? K(f16_tag) : K(bf16_tag), a, team, (hipStream_t)stream);
#undef K
}
