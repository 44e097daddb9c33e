// Root-mean-square norm of rows, behind the residual's addition, and its gradients.
//
//    h = x + residual (rounded to the rows' type, and kept);  y = h r w,  r = 1 / sqrt(mean(h^2) + eps)
//    dx = r (g - h r^2 mean(g h)) + dh with g = dy w;  dw = sum over rows of dy h r
//
// Sums are fp32.  h is rounded before the norm, so that the gradients, which have nothing but the h that
// was kept, are those of the y that was returned; y is rounded once.  r is computed again in the backward
// pass: its sum of squares rides along with that of g h.
//
// y may leave in 8 bits: e4m3 codes with one fp32 scale a row, amax / 448, that multiplies them (1 where that
// is no normal number).  The codes are taken from the fp32 y: one rounding.
#include "tftq_rows.h"

struct NormArgs {
    uint64_t x, residual, weight, y, h, codes, scales;  // residual, weight, h: 0 for none; codes and scales for 8 bits, else y
    int64_t x_stride, residual_stride;                  // bytes from row to row; all others are contiguous
    int64_t row0, rows;
    int cols, wide;  // wide: the weight is fp32 and the rows are not
    float eps, inv_cols;
};

// The weight's elements that belong to a vector: loaded early, widened late.
template <class T>
struct Weights {
    u32x4 raw, more;
    DEV void fetch(uint64_t weight, int wide, int col, int cols)
    {
        constexpr int EPV = Elem<T>::EPV;
        more = u32x4{0, 0, 0, 0};
        if (!weight) return;
        if (EPV == 8 && wide) {
            raw = fetch_row<4, false>(weight, col, cols);
            more = fetch_row<4, false>(weight, col + 4, cols);
        } else raw = fetch_row<Elem<T>::ESZ, false>(weight, col, cols);
    }
    DEV void settle(uint64_t weight, int wide, int col, int cols)
    {
        if (!weight) return;
        if (Elem<T>::EPV == 8 && wide) {
            raw = settle_row<4>(raw, col, cols);
            more = settle_row<4>(more, col + 4, cols);
        } else raw = settle_row<Elem<T>::ESZ>(raw, col, cols);
    }
    DEV void unpack(uint64_t weight, int wide, float (&w)[Elem<T>::EPV]) const
    {
        constexpr int EPV = Elem<T>::EPV;
        if (!weight) {
#pragma unroll
            for (int i = 0; i < EPV; i++) w[i] = 1.0f;
        } else if (EPV == 8 && wide) {
#pragma unroll
            for (int i = 0; i < EPV; i++) w[i] = as_f(i < 4 ? raw[i & 3] : more[i & 3]);
        } else Elem<T>::unpack(raw, w);
    }
};

DEV float inverse_root(float mean_square, float eps) { return 1.0f / __builtin_sqrtf(mean_square + eps); }

// One team of TEAM lanes to a row, which stays in its registers: memory is read and written once.
template <class T, int TEAM, int NV, bool FP8>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void k_rms_norm(const NormArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = TEAM > 256 ? 1 : 256 / TEAM;
    // weights in the registers of the residual, so that two workgroups of long rows run on a compute unit
    constexpr bool LATE = TEAM * NV >= 2048;
    __shared__ float lds[TEAM > 64 ? TEAM / 64 : 1];
    const int lane = threadIdx.x % TEAM;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (row >= a.rows) return;  // a whole team; teams of several wavefronts are whole workgroups
    const uint64_t px = a.x + (uint64_t)(row * a.x_stride), pr = a.residual + (uint64_t)(row * a.residual_stride);
    const uint64_t at = (uint64_t)(row * a.cols) * ESZ;

    u32x4 raw[NV], res[NV];
    Weights<T> weights[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) raw[v] = fetch_row<ESZ>(px, (v * TEAM + lane) * EPV, a.cols);
    if (a.residual) {
#pragma unroll
        for (int v = 0; v < NV; v++) res[v] = fetch_row<ESZ>(pr, (v * TEAM + lane) * EPV, a.cols);
    }
    auto fetch_weights = [&] {
#pragma unroll
        for (int v = 0; v < NV; v++) weights[v].fetch(a.weight, a.wide, (v * TEAM + lane) * EPV, a.cols);
    };
    if (!LATE) fetch_weights();
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int col = (v * TEAM + lane) * EPV;
        float f[EPV];
        raw[v] = settle_row<ESZ>(raw[v], col, a.cols);
        Elem<T>::unpack(raw[v], f);
        if (a.residual) {
            float r[EPV];
            Elem<T>::unpack(settle_row<ESZ>(res[v], col, a.cols), r);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] += r[i];
            raw[v] = Elem<T>::pack(f);
            store_row<ESZ>(a.h + at, col, a.cols, raw[v]);
            Elem<T>::unpack(raw[v], f);
        }
#pragma unroll
        for (int i = 0; i < EPV; i++) sum = __builtin_fmaf(f[i], f[i], sum);
    }
    if (LATE) fetch_weights();
    const float r = inverse_root(team_sum<TEAM>(sum, lds) * a.inv_cols, a.eps);
#pragma unroll
    for (int v = 0; v < NV; v++) weights[v].settle(a.weight, a.wide, (v * TEAM + lane) * EPV, a.cols);
    if constexpr (!FP8) {
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float f[EPV], w[EPV];
            Elem<T>::unpack(raw[v], f);
            weights[v].unpack(a.weight, a.wide, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] = f[i] * r * w[i];
            store_row<ESZ>(a.y + at, (v * TEAM + lane) * EPV, a.cols, Elem<T>::pack(f));
        }
    } else {
        float amax = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float f[EPV], w[EPV];
            Elem<T>::unpack(raw[v], f);
            weights[v].unpack(a.weight, a.wide, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) amax = fmaxf(amax, __builtin_fabsf(f[i] * r * w[i]));
        }
        amax = team_largest<TEAM>(amax, lds);
        const float part = amax / 448.0f, scale = part >= 0x1p-126f ? part : 1.0f, inverse = 1.0f / scale;
        if (lane == 0) as_global<float>(a.scales)[row] = scale;
        const uint64_t codes = a.codes + (uint64_t)(row * a.cols);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int col = (v * TEAM + lane) * EPV;
            float f[EPV], w[EPV];
            Elem<T>::unpack(raw[v], f);
            weights[v].unpack(a.weight, a.wide, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] = f[i] * r * w[i] * inverse;
            u32 c[2] = {pack_fp8x4(f[0], f[1], f[2], f[3]), 0};
            if constexpr (EPV == 8) c[1] = pack_fp8x4(f[4], f[5], f[6], f[7]);
            if (col + EPV <= a.cols) {
                if constexpr (EPV == 8) *as_global<u32x2_a1>(codes + (u32)col) = u32x2{c[0], c[1]};
                else *as_global<u32_a1>(codes + (u32)col) = c[0];
            } else {
#pragma unroll
                for (int i = 0; i < EPV; i++)
                    if (col + i < a.cols) as_global<uint8_t>(codes + (u32)col)[i] = (uint8_t)(c[i / 4] >> (i % 4 * 8));
            }
        }
    }
}

// Rows too long for the registers of a workgroup: its 1024 lanes go over the row two or three times, behind the
// first time in h (or x), which the caches may still have.
template <class T, bool FP8>
__global__ __launch_bounds__(1024) void k_rms_norm_long(const NormArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, STEP = 1024 * EPV;
    __shared__ float lds[16];
    const int64_t row = a.row0 + blockIdx.x;
    const uint64_t px = a.x + (uint64_t)(row * a.x_stride), pr = a.residual + (uint64_t)(row * a.residual_stride);
    const uint64_t at = (uint64_t)(row * a.cols) * ESZ, again = a.residual ? a.h + at : px;
    float sum = 0.0f;
    for (int col = threadIdx.x * EPV; col < a.cols; col += STEP) {
        u32x4 raw = load_row<ESZ, false>(px, col, a.cols);
        float f[EPV];
        Elem<T>::unpack(raw, f);
        if (a.residual) {
            float r[EPV];
            Elem<T>::unpack(load_row<ESZ>(pr, col, a.cols), r);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] += r[i];
            raw = Elem<T>::pack(f);
            store_row<ESZ, false>(a.h + at, col, a.cols, raw);
            Elem<T>::unpack(raw, f);
        }
#pragma unroll
        for (int i = 0; i < EPV; i++) sum = __builtin_fmaf(f[i], f[i], sum);
    }
    const float r = inverse_root(team_sum<1024>(sum, lds) * a.inv_cols, a.eps);
    // every lane reads back what it wrote itself: its own stores come before its own loads
    float inverse = 1.0f;
    for (int pass = FP8 ? 0 : 1; pass < 2; pass++) {
        float amax = 0.0f;
        for (int col = threadIdx.x * EPV; col < a.cols; col += STEP) {
            float f[EPV], w[EPV];
            Elem<T>::unpack(load_row<ESZ, false>(again, col, a.cols), f);
            Weights<T> weights;
            weights.fetch(a.weight, a.wide, col, a.cols);
            weights.settle(a.weight, a.wide, col, a.cols);
            weights.unpack(a.weight, a.wide, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] = f[i] * r * w[i];
            if (!FP8) store_row<ESZ>(a.y + at, col, a.cols, Elem<T>::pack(f));
            else if (pass == 0) {
#pragma unroll
                for (int i = 0; i < EPV; i++) amax = fmaxf(amax, __builtin_fabsf(f[i]));
            } else {
                const uint64_t codes = a.codes + (uint64_t)(row * a.cols);
#pragma unroll
                for (int i = 0; i < EPV; i++)
                    if (col + i < a.cols)
                        as_global<uint8_t>(codes + (u32)col)[i] = (uint8_t)pack_fp8x4(f[i] * inverse, 0.0f, 0.0f, 0.0f);
            }
        }
        if (FP8 && pass == 0) {
            amax = team_largest<1024>(amax, lds);
            const float part = amax / 448.0f, scale = part >= 0x1p-126f ? part : 1.0f;
            inverse = 1.0f / scale;
            if (threadIdx.x == 0) as_global<float>(a.scales)[row] = scale;
        }
    }
}

struct NormBackwardArgs {
    uint64_t dy, dh, h, weight, dx, sums;  // dh, weight, sums: 0 for none
    int64_t h_stride;                      // bytes; all others are contiguous
    int64_t rows;
    int cols, wide;
    float eps, inv_cols;
};

// A team goes over every (teams in the grid)-th row, one after the other, and keeps its part of dw in registers;
// a workgroup's teams add theirs up in LDS and leave a row of fp32 sums, which k_column_sums adds up.
template <class T, int TEAM, int NV>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void k_rms_norm_backward(const NormBackwardArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = TEAM > 256 ? 1 : 256 / TEAM;
    __shared__ float lds[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    __shared__ float add[TEAMS > 1 ? 256 * NV * EPV : 1];
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    float acc[NV][EPV];
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
        for (int i = 0; i < EPV; i++) acc[v][i] = 0.0f;
    Weights<T> weights[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) weights[v].fetch(a.weight, a.wide, (v * TEAM + lane) * EPV, a.cols);

    // the next row is on its way while this one is worked on, where there are registers for it
    constexpr bool AHEAD = TEAM * NV * EPV <= 8192;
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    u32x4 dy_next[NV], h_next[NV], dh_next[NV];
    auto fetch = [&](int64_t row) {
        const bool there = row < a.rows;
        const uint64_t at = (uint64_t)(row * a.cols) * ESZ, ph = a.h + (uint64_t)(row * a.h_stride);
        const int cols = there ? a.cols : 0;
#pragma unroll
        for (int v = 0; v < NV; v++) dy_next[v] = fetch_row<ESZ>(a.dy + at, (v * TEAM + lane) * EPV, cols);
#pragma unroll
        for (int v = 0; v < NV; v++) h_next[v] = fetch_row<ESZ>(ph, (v * TEAM + lane) * EPV, cols);
        if (a.dh) {
#pragma unroll
            for (int v = 0; v < NV; v++) dh_next[v] = fetch_row<ESZ>(a.dh + at, (v * TEAM + lane) * EPV, cols);
        }
    };
    int64_t row = (int64_t)blockIdx.x * TEAMS + team;
    if (AHEAD) fetch(row);
#pragma unroll
    for (int v = 0; v < NV; v++) weights[v].settle(a.weight, a.wide, (v * TEAM + lane) * EPV, a.cols);
    for (; row < a.rows; row += step) {
        if (!AHEAD) fetch(row);
        const uint64_t at = (uint64_t)(row * a.cols) * ESZ;
        u32x4 dy[NV], h[NV], dh[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            dy[v] = settle_row<ESZ>(dy_next[v], (v * TEAM + lane) * EPV, a.cols);
            h[v] = settle_row<ESZ>(h_next[v], (v * TEAM + lane) * EPV, a.cols);
            if (a.dh) dh[v] = settle_row<ESZ>(dh_next[v], (v * TEAM + lane) * EPV, a.cols);
        }
        if (AHEAD) fetch(row + step);
        float squares = 0.0f, along = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float f[EPV], g[EPV], w[EPV];
            Elem<T>::unpack(h[v], f);
            Elem<T>::unpack(dy[v], g);
            weights[v].unpack(a.weight, a.wide, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) {
                squares = __builtin_fmaf(f[i], f[i], squares);
                along = __builtin_fmaf(g[i] * w[i], f[i], along);
            }
        }
        team_sum2<TEAM>(squares, along, lds);
        const float r = inverse_root(squares * a.inv_cols, a.eps), c = r * r * (along * a.inv_cols);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float f[EPV], g[EPV], w[EPV], d[EPV];
            Elem<T>::unpack(h[v], f);
            Elem<T>::unpack(dy[v], g);
            weights[v].unpack(a.weight, a.wide, w);
            if (a.dh) Elem<T>::unpack(dh[v], d);
#pragma unroll
            for (int i = 0; i < EPV; i++) {
                acc[v][i] = __builtin_fmaf(g[i], f[i] * r, acc[v][i]);
                f[i] = r * (g[i] * w[i] - f[i] * c);
                if (a.dh) f[i] += d[i];
            }
            if (a.dx) store_row<ESZ>(a.dx + at, (v * TEAM + lane) * EPV, a.cols, Elem<T>::pack(f));
        }
    }
    if (!a.sums) return;
    const uint64_t sums = a.sums + (uint64_t)blockIdx.x * (uint64_t)a.cols * 4;
    if constexpr (TEAMS > 1) {
        constexpr int WIDTH = TEAM * EPV;
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int i = 0; i < EPV; i++) add[(team * NV + v) * WIDTH + i * TEAM + lane] = acc[v][i];
        __syncthreads();
        for (int c = threadIdx.x; c < NV * WIDTH; c += 256) {
            float s = 0.0f;
            for (int t = 0; t < TEAMS; t++) s += add[t * NV * WIDTH + c];
            const int v = c / WIDTH, i = c % WIDTH / TEAM, l = c % TEAM, col = (v * TEAM + l) * EPV + i;
            if (col < a.cols) as_global<float>(sums)[col] = s;
        }
    } else {
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int i = 0; i < EPV; i += 4)
                store_row<4, false>(sums, (v * TEAM + lane) * EPV + i, a.cols,
                                    u32x4{as_u(acc[v][i]), as_u(acc[v][i + 1]), as_u(acc[v][i + 2]), as_u(acc[v][i + 3])});
    }
}

// Rows too long for that: first r and c of every row, then dx and the sums, a workgroup to 256 vectors of columns
// and a share of the rows, four rows at a time.
template <class T>
__global__ __launch_bounds__(1024) void k_rms_norm_backward_long(const NormBackwardArgs a, uint64_t factors)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, U = 2, STEP = 1024 * EPV;
    __shared__ float lds[32];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t at = (uint64_t)(row * a.cols) * ESZ, ph = a.h + (uint64_t)(row * a.h_stride);
        float squares = 0.0f, along = 0.0f;
        for (int col = threadIdx.x * EPV; col < a.cols; col += U * STEP) {
            Weights<T> weights[U];
            u32x4 h[U], dy[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                h[u] = fetch_row<ESZ, false>(ph, col + u * STEP, a.cols);
                dy[u] = fetch_row<ESZ, false>(a.dy + at, col + u * STEP, a.cols);
                weights[u].fetch(a.weight, a.wide, col + u * STEP, a.cols);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                float f[EPV], g[EPV], w[EPV];
                weights[u].settle(a.weight, a.wide, col + u * STEP, a.cols);
                weights[u].unpack(a.weight, a.wide, w);
                Elem<T>::unpack(settle_row<ESZ>(h[u], col + u * STEP, a.cols), f);
                Elem<T>::unpack(settle_row<ESZ>(dy[u], col + u * STEP, a.cols), g);
#pragma unroll
                for (int i = 0; i < EPV; i++) {
                    squares = __builtin_fmaf(f[i], f[i], squares);
                    along = __builtin_fmaf(g[i] * w[i], f[i], along);
                }
            }
        }
        team_sum2<1024>(squares, along, lds);
        const float r = inverse_root(squares * a.inv_cols, a.eps);
        if (threadIdx.x < 2) as_global<float>(factors)[2 * row + threadIdx.x] = threadIdx.x ? r * r * (along * a.inv_cols) : r;
    }
}
template <class T>
__global__ __launch_bounds__(256) void k_rms_norm_backward_columns(const NormBackwardArgs a, uint64_t factors)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, U = 4;
    const int col = (int)(blockIdx.x * 256 + threadIdx.x) * EPV;
    if (col >= a.cols) return;
    float acc[EPV] = {}, w[EPV];
    Weights<T> weights;
    weights.fetch(a.weight, a.wide, col, a.cols);
    weights.settle(a.weight, a.wide, col, a.cols);
    weights.unpack(a.weight, a.wide, w);
    for (int64_t first = (int64_t)blockIdx.y * U; first < a.rows; first += (int64_t)gridDim.y * U) {
        u32x4 h[U], dy[U], dh[U];
        float r[U], c[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t row = first + u < a.rows ? first + u : a.rows - 1;
            const uint64_t at = (uint64_t)(row * a.cols) * ESZ;
            h[u] = fetch_row<ESZ>(a.h + (uint64_t)(row * a.h_stride), col, a.cols);
            dy[u] = fetch_row<ESZ>(a.dy + at, col, a.cols);
            if (a.dh) dh[u] = fetch_row<ESZ>(a.dh + at, col, a.cols);
            r[u] = as_global<const float>(factors)[2 * row];
            c[u] = as_global<const float>(factors)[2 * row + 1];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (first + u >= a.rows) continue;
            float f[EPV], g[EPV], d[EPV];
            Elem<T>::unpack(settle_row<ESZ>(h[u], col, a.cols), f);
            Elem<T>::unpack(settle_row<ESZ>(dy[u], col, a.cols), g);
            if (a.dh) Elem<T>::unpack(settle_row<ESZ>(dh[u], col, a.cols), d);
#pragma unroll
            for (int i = 0; i < EPV; i++) {
                acc[i] = __builtin_fmaf(g[i], f[i] * r[u], acc[i]);
                f[i] = r[u] * (g[i] * w[i] - f[i] * c[u]);
                if (a.dh) f[i] += d[i];
            }
            if (a.dx) store_row<ESZ>(a.dx + (uint64_t)((first + u) * a.cols) * ESZ, col, a.cols, Elem<T>::pack(f));
        }
    }
    if (!a.sums) return;
#pragma unroll
    for (int i = 0; i < EPV; i += 4)
        store_row<4, false>(a.sums + (uint64_t)blockIdx.y * (uint64_t)a.cols * 4, col + i, a.cols,
                            u32x4{as_u(acc[i]), as_u(acc[i + 1]), as_u(acc[i + 2]), as_u(acc[i + 3])});
}

// out[c] = the sum of sums[p][c] over p, rounded once: 4 lanes to 16 columns, 64 of the parts side by side.
template <class T>
__global__ __launch_bounds__(256) void k_column_sums(uint64_t sums, int64_t parts, int cols, uint64_t out)
{
    __shared__ float add[64][17];
    const int lane = threadIdx.x & 3, group = threadIdx.x >> 2, col = (int)blockIdx.x * 16 + lane * 4;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int64_t p = group; p < parts; p += 64) {
        const u32x4 v = load_row<4, false>(sums + (uint64_t)p * (uint64_t)cols * 4, col, cols);
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] += as_f(v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) add[group][lane * 4 + i] = s[i];
    __syncthreads();
    // 16 threads to a column, then one
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const float part = (add[g][c] + add[g + 16][c]) + (add[g + 32][c] + add[g + 48][c]);
    __syncthreads();
    add[g][c] = part;
    __syncthreads();
    if (threadIdx.x >= 16) return;
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) total += add[i][c];
    const int64_t at = (int64_t)blockIdx.x * 16 + c;
    if (at < cols) Elem<T>::store(out, at, total);
}

// The values of 8-bit rows, a lane for EPV of them.
template <class T, int TEAM>
__global__ __launch_bounds__(256) void k_fp8_rows(uint64_t codes, uint64_t scales, int64_t row0, int64_t rows, int cols, uint64_t out)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, U = 2;
    const int64_t row = row0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (row >= rows) return;
    const float scale = as_global<const float>(scales)[row];
    const uint64_t from = codes + (uint64_t)(row * cols), to = out + (uint64_t)(row * cols) * ESZ;
    for (int col = threadIdx.x % TEAM * EPV; col < cols; col += U * TEAM * EPV) {
        u32 w[U][2];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = col + u * TEAM * EPV;
            w[u][0] = w[u][1] = 0;
            if (at + EPV <= cols) {
                if constexpr (EPV == 8) {
                    const u32x2 v = LOAD_STREAM(as_global<const u32x2_a1>(from + (u32)at));
                    w[u][0] = v.x;
                    w[u][1] = v.y;
                } else w[u][0] = LOAD_STREAM(as_global<const u32_a1>(from + (u32)at));
            } else {
#pragma unroll
                for (int i = 0; i < EPV; i++)
                    if (at + i < cols) w[u][i / 4] |= (u32)as_global<const uint8_t>(from + (u32)at)[i] << (i % 4 * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float f[EPV];
#pragma unroll
            for (int i = 0; i < EPV; i += 4) {
                float four[4];
                unpack_fp8x4(w[u][i / 4], four);
#pragma unroll
                for (int j = 0; j < 4; j++) f[i + j] = four[j] * scale;
            }
            store_row<ESZ>(to, col + u * TEAM * EPV, cols, Elem<T>::pack(f));
        }
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Lanes and vectors to a row of `vectors`; {0, 0}: too long for registers.  Two vectors a lane hide more of memory's latency
// than one, and lanes that a row leaves idle cost as much as others: rows of 16 vectors (163840 fp16) take 17.5 us with 8 lanes of
// two, 18.4 with 16, 47 with 64; rows of 512 (8192 bf16 with a residual) 45.8 with 512 lanes, 47.5 with 256 of two, one
// row 3.4 and 3.8.
static RowShape norm_shape(int64_t vectors)
{
    if (vectors <= 8) return {8, 1};
    if (vectors <= 16) return {8, 2};
    if (vectors <= 32) return {16, 2};
    if (vectors <= 64) return {32, 2};
    if (vectors <= 128) return {64, 2};
    if (vectors <= 256) return {256, 1};
    if (vectors <= 512) return {512, 1};
    if (vectors <= 1024) return {512, 2};
    if (vectors <= 2048) return {1024, 2};
    if (vectors <= 4096) return {1024, 4};
    return {0, 0};
}

// The same for the backward pass, whose lanes keep a column's sum and the next row beside: us of rows of 42
// vectors (65536 bf16) 42.3 with 16 lanes of three, 47.2 with 64 of one; of 251 (8192 fp32) 30.0 with 64 of four, 42.1 with
// 256 of one; of 256 (16384 bf16, where four take all registers) 58.2 and 51.9; of 512 (8192 bf16) 49.9 with 512 of
// one, 52.9 with 256 of two.
static RowShape norm_backward_shape(int64_t vectors, int size)
{
    if (vectors <= 8) return {8, 1};
    if (vectors <= 16) return {8, 2};
    if (vectors <= 32) return {16, 2};
    if (vectors <= 48) return {16, 3};
    if (vectors <= 64) return {32, 2};
    if (vectors <= 128) return {64, 2};
    if (vectors <= 192) return {64, 3};
    if (vectors <= 256) return size == 4 ? RowShape{64, 4} : RowShape{256, 1};
    if (vectors <= 512) return {512, 1};
    if (vectors <= 1024) return {512, 2};
    if (vectors <= 2048) return {512, 4};
    return {0, 0};
}

#define SHAPE(TEAM, NV) case TEAM * 16 + NV: K(TEAM, NV); break;

template <class T, bool FP8>
static int norm(NormArgs a, hipStream_t st)
{
    const RowShape shape = norm_shape((a.cols + Elem<T>::EPV - 1) / Elem<T>::EPV);
    const void *k = (const void *)k_rms_norm_long<T, FP8>;
#define K(TEAM, NV) k = (const void *)k_rms_norm<T, TEAM, NV, FP8>
    switch (shape.team * 16 + shape.nv) {
        SHAPE(8, 1) SHAPE(8, 2) SHAPE(16, 2) SHAPE(32, 2) SHAPE(64, 2) SHAPE(256, 1) SHAPE(512, 1) SHAPE(512, 2) SHAPE(1024, 2) SHAPE(1024, 4)
    }
#undef K
    const int threads = shape.team == 0 ? 1024 : shape.team > 256 ? shape.team : 256, teams = shape.team == 0 ? 1 : threads / shape.team;
    const int64_t at_once = ROWS_THREADS / threads * teams;
    for (a.row0 = 0; a.row0 < a.rows; a.row0 += at_once) {
        const int64_t left = std::min(at_once, a.rows - a.row0);
        void *args[] = {(void *)&a};
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)((left + teams - 1) / teams)), dim3(threads), args, 0, st)) return rc;
    }
    return 0;
}

// Workgroups of the backward kernels, whose sums k_column_sums adds up: as many as run at once with their registers, so that
// none starts when the others end, and no more sums than that (8192 rows of 4096 bf16 49.9 us with 256, 52.8 with 512, 58.2
// with 1024).
static int64_t norm_parts(int64_t rows, int64_t cols, int size)
{
    const RowShape shape = norm_backward_shape((cols * size + 15) / 16, size);
    const int64_t teams = shape.team == 0 || shape.team > 256 ? 1 : 256 / shape.team;
    int64_t most = shape.team > 256 ? 256 : 512;
    if (shape.team == 0) most = std::max<int64_t>(1, 1280 / ((cols * size + 4095) / 4096));  // five for every compute unit
    return std::min(most, (rows + teams - 1) / teams);
}

template <class T>
static int norm_backward(NormBackwardArgs a, uint64_t factors, int64_t parts, hipStream_t st)
{
    const RowShape shape = norm_backward_shape((a.cols + Elem<T>::EPV - 1) / Elem<T>::EPV, Elem<T>::ESZ);
    if (shape.team == 0) {
        void *args[] = {(void *)&a, (void *)&factors};
        int rc = (int)hipLaunchKernel((const void *)k_rms_norm_backward_long<T>, dim3((unsigned)std::min<int64_t>(a.rows, 2048)), dim3(1024),
                                      args, 0, st);
        if (rc) return rc;
        const unsigned across = (unsigned)((a.cols + 256 * Elem<T>::EPV - 1) / (256 * Elem<T>::EPV));
        return (int)hipLaunchKernel((const void *)k_rms_norm_backward_columns<T>, dim3(across, (unsigned)parts), dim3(256), args, 0, st);
    }
    const void *k = nullptr;
#define K(TEAM, NV) k = (const void *)k_rms_norm_backward<T, TEAM, NV>
    if constexpr (Elem<T>::ESZ == 4) {
        if (shape.team == 64 && shape.nv == 4) K(64, 4);
    } else if (shape.team == 256) K(256, 1);
    switch (shape.team * 16 + shape.nv) {
        SHAPE(8, 1) SHAPE(8, 2) SHAPE(16, 2) SHAPE(16, 3) SHAPE(32, 2) SHAPE(64, 2) SHAPE(64, 3) SHAPE(512, 1) SHAPE(512, 2) SHAPE(512, 4)
    }
#undef K
#undef SHAPE
    void *args[] = {(void *)&a};
    return (int)hipLaunchKernel(k, dim3((unsigned)parts), dim3(shape.team > 256 ? shape.team : 256), args, 0, st);
}

extern "C" int tftq_rms_norm(int dtype, int weight_dtype, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                             const void *weight, int64_t rows, int64_t cols, float eps, void *h, void *y, void *codes, float *scales,
                             int device, void *stream)
{
    if (!dtype_ok(dtype) || (weight && weight_dtype != dtype && weight_dtype != TFTQ_F32)) return TFTQ_E_DTYPE;
    if (!rows_ok(rows, cols)) return TFTQ_E_SHAPE;
    if (rows == 0 || cols == 0) return 0;
    if (!x || !residual != !h || !codes != !scales || !y == !codes || !(eps >= 0.0f)) return TFTQ_E_ARG;
    const int64_t across = rows > 1 ? cols : 0;
    if (x_stride < across || (residual && residual_stride < across)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const int size = dtype_size(dtype);
    const NormArgs a = {(uint64_t)x, (uint64_t)residual, (uint64_t)weight, (uint64_t)y, (uint64_t)h, (uint64_t)codes, (uint64_t)scales,
                        x_stride * size, residual_stride * size, 0, rows, (int)cols, weight && weight_dtype != dtype, eps, 1.0f / (float)cols};
    hipStream_t st = (hipStream_t)stream;
    if (codes) return dtype == TFTQ_F32 ? norm<float, true>(a, st) : dtype == TFTQ_F16 ? norm<f16_tag, true>(a, st) : norm<bf16_tag, true>(a, st);
    return dtype == TFTQ_F32 ? norm<float, false>(a, st) : dtype == TFTQ_F16 ? norm<f16_tag, false>(a, st) : norm<bf16_tag, false>(a, st);
}

extern "C" int64_t tftq_rms_norm_backward_workspace(int dtype, int64_t rows, int64_t cols)
{
    if (!dtype_ok(dtype)) return TFTQ_E_DTYPE;
    if (!rows_ok(rows, cols)) return TFTQ_E_SHAPE;
    if (rows == 0 || cols == 0) return 0;
    return norm_parts(rows, cols, dtype_size(dtype)) * cols * 4 + rows * 8;
}

extern "C" int tftq_rms_norm_backward(int dtype, int weight_dtype, const void *dy, const void *dh, const void *h, int64_t h_stride,
                                      const void *weight, int64_t rows, int64_t cols, float eps, void *dx, void *dweight, void *workspace,
                                      int64_t workspace_bytes, int device, void *stream)
{
    if (!dtype_ok(dtype) || (weight && weight_dtype != dtype && weight_dtype != TFTQ_F32)) return TFTQ_E_DTYPE;
    if (!rows_ok(rows, cols)) return TFTQ_E_SHAPE;
    if (cols == 0 || (rows == 0 && !dweight)) return 0;
    if ((dweight && !weight) || (rows && (!dy || !h || !workspace || ((uintptr_t)workspace & 15))) || (!dx && !dweight) || !(eps >= 0.0f)) return TFTQ_E_ARG;
    if (rows && h_stride < (rows > 1 ? cols : 0)) return TFTQ_E_ARG;
    const int size = dtype_size(dtype);
    const int64_t parts = rows ? norm_parts(rows, cols, size) : 0, sums = parts * cols * 4;
    if (rows && workspace_bytes < sums + rows * 8) return TFTQ_E_SIZE;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    hipStream_t st = (hipStream_t)stream;
    if (rows) {
        const NormBackwardArgs a = {(uint64_t)dy, (uint64_t)dh, (uint64_t)h, (uint64_t)weight, (uint64_t)dx, dweight ? (uint64_t)workspace : 0,
                                    h_stride * size, rows, (int)cols, weight && weight_dtype != dtype, eps, 1.0f / (float)cols};
        const uint64_t factors = (uint64_t)workspace + (uint64_t)sums;
        const int rc = dtype == TFTQ_F32   ? norm_backward<float>(a, factors, parts, st)
                       : dtype == TFTQ_F16 ? norm_backward<f16_tag>(a, factors, parts, st)
                                           : norm_backward<bf16_tag>(a, factors, parts, st);
        if (rc || !dweight) return rc;
    }
    uint64_t from = (uint64_t)workspace, to = (uint64_t)dweight;
    int64_t p = parts;
    int c = (int)cols;
    void *args[] = {(void *)&from, (void *)&p, (void *)&c, (void *)&to};
    const void *k = weight_dtype == TFTQ_F32   ? (const void *)k_column_sums<float>
                    : weight_dtype == TFTQ_F16 ? (const void *)k_column_sums<f16_tag>
                                               : (const void *)k_column_sums<bf16_tag>;
    return (int)hipLaunchKernel(k, dim3((unsigned)((cols + 15) / 16)), dim3(256), args, 0, st);
}

extern "C" int tftq_fp8_rows_dequantize(int dtype, const void *codes, const float *scales, int64_t rows, int64_t cols, void *out, int device,
                                        void *stream)
{
    if (!dtype_ok(dtype)) return TFTQ_E_DTYPE;
    if (!rows_ok(rows, cols)) return TFTQ_E_SHAPE;
    if (rows == 0 || cols == 0) return 0;
    if (!codes || !scales || !out) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const int64_t vectors = (cols * dtype_size(dtype) + 15) / 16, team = vectors <= 16 ? 8 : vectors <= 128 ? 64 : 256, teams = 256 / team;
    uint64_t from = (uint64_t)codes, by = (uint64_t)scales, to = (uint64_t)out;
    int64_t row0 = 0;
    int c = (int)cols;
    void *args[] = {(void *)&from, (void *)&by, (void *)&row0, (void *)&rows, (void *)&c, (void *)&to};
#define K(T) (team == 8 ? (const void *)k_fp8_rows<T, 8> : team == 64 ? (const void *)k_fp8_rows<T, 64> : (const void *)k_fp8_rows<T, 256>)
    const void *k = dtype == TFTQ_F32 ? K(float) : dtype == TFTQ_F16 ? K(f16_tag) : K(bf16_tag);
#undef K
    const int64_t at_once = ROWS_THREADS / team;
    for (; row0 < rows; row0 += at_once)
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)((std::min(at_once, rows - row0) + teams - 1) / teams)), dim3(256), args, 0, (hipStream_t)stream))
            return rc;
    return 0;
}
