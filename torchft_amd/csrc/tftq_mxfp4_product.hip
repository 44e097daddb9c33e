// The product of two 4-bit microscaled matrices, c[i][j] = sum_k a[i][k] b[j][k], and its C entry.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "tftq_mxfp4.h"

// A result as it is stored.
template <int DTYPE>
struct MxOut {
    static constexpr int SIZE = DTYPE == TFTQ_F32 ? 4 : 2, V = 16 / SIZE;
    typedef _Float16 H2 __attribute__((ext_vector_type(2)));
    typedef __bf16 B2 __attribute__((ext_vector_type(2)));
    __device__ static uint32_t two(float a, float b)
    {
        if constexpr (DTYPE == TFTQ_F16) return __builtin_bit_cast(uint32_t, H2{(_Float16)a, (_Float16)b});
        else return __builtin_bit_cast(uint32_t, B2{(__bf16)a, (__bf16)b});
    }
    __device__ static void put(uint8_t *out, int64_t at, float v)
    {
        if constexpr (DTYPE == TFTQ_F32) ((float *)out)[at] = v;
        else if constexpr (DTYPE == TFTQ_F16) ((_Float16 *)out)[at] = (_Float16)v;
        else ((__bf16 *)out)[at] = (__bf16)v;
    }
};

// The product in tiles (tftq_tile.h), as many workgroups as the units hold at once, each with its tiles one after
// the other: a tile's first panels come while the last one's values go out, which is worth 7 % at 2048
// columns.  Bound by the matrix cores at the clock that the card's power allows: 8192x14336x4096 to bf16
// 221 us (4.35 PFLOP/s), 8192x4096x14336 206 us (4.7, what the loop alone reaches on long sums),
// 2048x2048x2048 10.5 us.
template <class T, int DTYPE>
__global__ __launch_bounds__(T::THREADS) void k_mx_product(TileOperand a, TileOperand b, int panels, uint8_t *out, int64_t ld,
                                                           int tiles_m, int tiles_n)
{
    __shared__ __attribute__((aligned(128))) uint8_t lds[T::LDS_PIECES];
    using O = MxOut<DTYPE>;
    int apart, pieces;
    const int first = tile_pieces(blockIdx.x, gridDim.x, tiles_m * tiles_n, &apart, &pieces);
    auto place = [&](int n, int *row0, int *col0) {
        int tm, tn;
        tile_place(first + n * apart, tiles_m, tiles_n, &tm, &tn);
        *row0 = tm * T::ROWS, *col0 = tn * T::COLS;
    };
    T t;
    t.multiply(TilePair{a, b}, panels, pieces, place, lds, [&](int row0, int col0) {
        t.template store_pieces<O::SIZE>(row0, col0, lds + T::PIECES_AT, O::two, [&](tile_i4 v, int row, int col) {
            if (row >= a.rows) return;
            uint8_t *at = out + ((int64_t)row * ld + col) * O::SIZE;
            if (col + O::V <= b.rows) {  // at any element's address
                *(mx_u4_any *)at = __builtin_bit_cast(mx_u4, v);
                return;
            }
#pragma unroll
            for (int n = 0; n < O::V; n++) {
                if (col + n >= b.rows) return;
                if constexpr (O::SIZE == 4) ((int *)at)[n] = v[n];
                else ((uint16_t *)at)[n] = (uint16_t)(v[n / 2] >> (16 * (n & 1)));
            }
        });
    });
}

// Few rows times a matrix, out[i][j] = sum_k Q(x)[i][k] b[j][k]: the tokens of a model that is served.  The
// time is that of b's bytes: a workgroup takes 16 rows of b, its 8 wavefronts share the panels between
// them with two panels' loads on the way, and their sums are added in LDS, always in the same order.
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 32 codes of row lane % 16 from quarter lane / 16 of 64 bytes.
// X: the type of x, which the workgroup quantises into LDS while its first loads are on the way (every
// workgroup all of x: what that costs against a launch of its own, few_rows); MxQuantized: x's codes lie
// in panels.  TOKENS: groups of 16 rows of x.  14336x4096, one row of bf16:
// 7.4 us (31 MB, 4.2 TB/s, the launch in it).
constexpr int FEW_WAVES = 8, FEW_PITCH = PANEL_BYTES + 16;  // a token's codes of a panel, its scales and padding
constexpr int FEW_SUMS = FEW_WAVES * 16 * 20 * 4;           // a group's sums of every wavefront
constexpr int FEW_MOST = 64;                                // rows of x
constexpr int64_t FEW_WIDEST = 1 << 26;                     // rows of b: a launch has fewer than 2^32 threads
struct MxQuantized {};

template <class X>
__device__ static inline void few_quantize(const uint8_t *x, int64_t ld, int rows, int cols, uint8_t *tokens)
{
    const int blocks = (cols + 255) / 256 * 8;
    for (int id = threadIdx.x; id < rows * blocks; id += 64 * FEW_WAVES) {
        const int i = id / blocks, block = id - i * blocks;
        constexpr int VECTORS = 32 / X::V;
        mx_u4 v[VECTORS];
        uint32_t m = 0;
#pragma unroll
        for (int n = 0; n < VECTORS; n++) v[n] = mx_read<X>(x + i * ld * X::SIZE, block * 32 + n * X::V, cols);
#pragma unroll
        for (int n = 0; n < VECTORS; n++)
#pragma unroll
            for (int w = 0; w < 4; w++) m = X::mag_max(m, X::mag(v[n][w]));
        const uint32_t byte = mx_byte(X::bits(X::mag_all(m)));
        const float scale = mx_scale(byte);
        mx_u4 c;
#pragma unroll
        for (int n = 0; n < 4; n++)
            c[n] = X::SIZE == 2 ? mx_codes<X>(v[n], scale) : mx_codes<X>(v[2 * n % VECTORS], scale) | mx_codes<X>(v[(2 * n + 1) % VECTORS], scale) << 16;
        uint8_t *to = tokens + ((block >> 3) * rows + i) * FEW_PITCH;
        *(mx_u4 *)(to + (block & 7) * 16) = c;
        to[PANEL_BYTES + (block & 7)] = (uint8_t)byte;
    }
    __syncthreads();
}

template <class X, int DTYPE, int TOKENS>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_mx_few(const uint8_t *x, int64_t ld, const uint8_t *x_scales, int rows, TileOperand b,
                                                           int cols, uint8_t *out, int64_t ld_out)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr bool READY = std::is_same<X, MxQuantized>::value;
    uint8_t *tokens = lds + FEW_SUMS;
    const int lane = threadIdx.x & 63, wave = tile_wave(), quarter = lane >> 4, panels = (cols + 255) >> 8;
    const int row0 = tile_piece(blockIdx.x, gridDim.x) * 16, row = min(row0 + (lane & 15), b.rows - 1);

    constexpr int AHEAD = 2;  // panels in flight
    struct Panel {
        tile_i4 b[2], x[READY ? 2 * TOKENS : 1];
        uint64_t b_scales, x_scales[READY ? TOKENS : 1];
    } ahead[AHEAD];
    auto load = [&](int s, Panel &p) {
        if (s >= panels) return;
        const uint8_t *from = b.panels + ((int64_t)s * b.rows + row) * PANEL_BYTES + quarter * 16;
        p.b[0] = *(const tile_i4 *)from, p.b[1] = *(const tile_i4 *)(from + 64);
        p.b_scales = *(const uint64_t *)(b.scales + ((int64_t)s * ((b.rows + 1) & ~1) + row) * 8);
        if constexpr (READY) {
#pragma unroll
            for (int g = 0; g < TOKENS; g++) {
                const int i = min(g * 16 + (lane & 15), rows - 1);
                const uint8_t *at = x + ((int64_t)s * rows + i) * PANEL_BYTES + quarter * 16;
                p.x[2 * g] = *(const tile_i4 *)at, p.x[2 * g + 1] = *(const tile_i4 *)(at + 64);
                p.x_scales[g] = *(const uint64_t *)(x_scales + ((int64_t)s * ((rows + 1) & ~1) + i) * 8);
            }
        }
    };
#pragma unroll
    for (int n = 0; n < AHEAD; n++) load(wave + n * FEW_WAVES, ahead[n]);
    if constexpr (!READY) few_quantize<X>(x, ld, rows, cols, tokens);

    tile_f4 acc[TOKENS] = {};
    auto multiply = [&](int s, const Panel &p) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const tile_i8 w = {p.b[h][0], p.b[h][1], p.b[h][2], p.b[h][3], 0, 0, 0, 0};
            const uint32_t sw = (uint32_t)(p.b_scales >> (32 * h)) >> (8 * quarter);
#pragma unroll
            for (int g = 0; g < TOKENS; g++) {
                tile_i4 d;
                uint32_t st;
                if constexpr (READY) {
                    d = p.x[2 * g + h], st = (uint32_t)(p.x_scales[g] >> (32 * h));
                } else {
                    const uint8_t *from = tokens + (s * rows + min(g * 16 + (lane & 15), rows - 1)) * FEW_PITCH;
                    d = *(const tile_i4 *)(from + h * 64 + quarter * 16), st = *(const uint32_t *)(from + PANEL_BYTES + 4 * h);
                }
                const tile_i8 t = {d[0], d[1], d[2], d[3], 0, 0, 0, 0};
                acc[g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, t, acc[g], 4, 4, 0, sw, 0, st >> (8 * quarter));
            }
        }
    };
    for (int s = wave; s < panels; s += AHEAD * FEW_WAVES) {
#pragma unroll
        for (int n = 0; n < AHEAD; n++) {
            if (s + n * FEW_WAVES >= panels) break;
            multiply(s + n * FEW_WAVES, ahead[n]);
            load(s + (n + AHEAD) * FEW_WAVES, ahead[n]);
        }
    }

    // a lane has rows 4 (lane / 16) to + 3 of b for token lane % 16
    float *sums = (float *)lds;
#pragma unroll
    for (int g = 0; g < TOKENS; g++) {
        *(tile_f4 *)(sums + (wave * 16 + (lane & 15)) * 20 + 4 * quarter) = acc[g];
        __syncthreads();
        const int i = threadIdx.x >> 4, j = threadIdx.x & 15;
        if (i < 16) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < FEW_WAVES; k++) v += sums[(k * 16 + i) * 20 + j];
            if (g * 16 + i < rows && row0 + j < b.rows) MxOut<DTYPE>::put(out, (int64_t)(g * 16 + i) * ld_out + row0 + j, v);
        }
        __syncthreads();
    }
}

template <class X, int DTYPE>
static int few(const uint8_t *x, int64_t ld, const uint8_t *x_scales, int rows, const TileOperand &b, int cols, uint8_t *out, int64_t ld_out,
               hipStream_t st)
{
    const bool ready = std::is_same<X, MxQuantized>::value;
    const unsigned lds = FEW_SUMS + (ready ? 0 : (unsigned)(rows * ((cols + 255) / 256) * FEW_PITCH)), groups = (unsigned)((b.rows + 15) / 16);
    void *args[] = {(void *)&x, (void *)&ld, (void *)&x_scales, (void *)&rows, (void *)&b, (void *)&cols, (void *)&out, (void *)&ld_out};
    const void *k = rows <= 16 ? (const void *)k_mx_few<X, DTYPE, 1> : rows <= 32 ? (const void *)k_mx_few<X, DTYPE, 2> : (const void *)k_mx_few<X, DTYPE, 4>;
    return (int)hipLaunchKernel(k, dim3(groups), dim3(64 * FEW_WAVES), args, lds, st);
}

// A launch of tiles of one size.
template <class T>
static int product(int dtype, const TileOperand &a, const TileOperand &b, int panels, uint8_t *out, int64_t ld, hipStream_t st)
{
    int tiles_m = (a.rows + T::ROWS - 1) / T::ROWS, tiles_n = (b.rows + T::COLS - 1) / T::COLS;
    if ((int64_t)tiles_m * tiles_n > INT_MAX) return TFTQ_E_SHAPE;  // 8.8e12 results or more
    void *args[] = {(void *)&a, (void *)&b, (void *)&panels, (void *)&out, (void *)&ld, (void *)&tiles_m, (void *)&tiles_n};
    const void *k = dtype == TFTQ_F32 ? (const void *)k_mx_product<T, TFTQ_F32>
                    : dtype == TFTQ_F16 ? (const void *)k_mx_product<T, TFTQ_F16>
                                        : (const void *)k_mx_product<T, TFTQ_BF16>;
    // as many workgroups as the 256 compute units hold at once; each takes its tiles one after the other
    const int resident = 256 * (160 * 1024 / T::LDS_PIECES), tiles = tiles_m * tiles_n;
    return (int)hipLaunchKernel(k, dim3((unsigned)(tiles < resident ? tiles : resident)), dim3(T::THREADS), args, 0, st);
}

extern "C" int tftq_mx_product(int dtype, const void *a, int64_t m, const void *b, int64_t n, int64_t k, void *out,
                               int64_t row_stride, int device, void *stream)
{
    if (dtype != TFTQ_F32 && dtype != TFTQ_F16 && dtype != TFTQ_BF16) return TFTQ_E_DTYPE;
    if (m < 0 || n < 0 || k < 0 || m > MX_MOST || n > MX_MOST || k > MX_MOST) return TFTQ_E_SHAPE;
    if (m == 0 || n == 0) return 0;
    if (!out || row_stride < (m > 1 ? n : 0)) return TFTQ_E_ARG;
    if (k > 0 && (!a || !b || (((uintptr_t)a | (uintptr_t)b) & 15))) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const MxMatrix ma = mx_matrix((void *)a, m, k), mb = mx_matrix((void *)b, n, k);
    const TileOperand ta = {ma.panels, ma.scales, (int)m}, tb = {mb.panels, mb.scales, (int)n};
    const int panels = (int)((k + 255) / 256);
    hipStream_t st = (hipStream_t)stream;
    // Up to 64 rows: by 16 rows of b and all of a (k_mx_few) up to 16 rows of a, and beyond that where tiles
    // of 64 x 64 are too few for the units: with the quantisation of a before it, n 14336, k 4096,
    // 24 rows 15.6 us (tiles 12.6), 64 rows 30.6 (12.9); n 4096, k 14336, 24 rows 14.8 (29.2), 64 rows
    // 23.6 (29.5); n 1024, k 4096, 64 rows 10.0 (11.6).
    if ((m <= 16 && n <= FEW_WIDEST) || (m <= FEW_MOST && (n + 63) / 64 < 160)) {
        switch (dtype) {
        case TFTQ_F32: return few<MxQuantized, TFTQ_F32>(ta.panels, 0, ta.scales, (int)m, tb, (int)k, (uint8_t *)out, row_stride, st);
        case TFTQ_F16: return few<MxQuantized, TFTQ_F16>(ta.panels, 0, ta.scales, (int)m, tb, (int)k, (uint8_t *)out, row_stride, st);
        default: return few<MxQuantized, TFTQ_BF16>(ta.panels, 0, ta.scales, (int)m, tb, (int)k, (uint8_t *)out, row_stride, st);
        }
    }
    const TileShape choice[] = {TILES_256, TILES_192X256, TILES_128, TILES_64_FP4};
    int best = 0;
    double least = 0;
    for (int i = 0; i < 4; i++) {
        const double count = (double)((m + choice[i].high - 1) / choice[i].high) * (double)((n + choice[i].wide - 1) / choice[i].wide);
        const double time = tile_time(choice[i], count, count * panels, panels);
        if (i == 0 || time < least) best = i, least = time;
    }
    switch (best) {
    case 0: return product<Tile<256, 256, 2, 4, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    case 1: return product<Tile<192, 256, 2, 4, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    case 2: return product<Tile<128, 128, 2, 2, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    default: return product<Tile<64, 64, 2, 2, true, 3>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    }
}

// Whether x [m, k] is quantised by the workgroups of the product with n rows.  That saves a launch and the
// wait for it, 2 to 3 us, and costs every workgroup time that grows with m k, which those that find no
// room at first add to: n 14336, k 4096, aligned rows: 1 row 6.9 us (two launches 10.1), 4 rows 8.4
// (10.8), 8 rows 11.0 (11.5), 16 rows 15.3 (12.6); n 1024: 1 row 3.4 (5.4), 16 rows 5.7 (6.3), 24 rows 7.3
// (7.2).  Rows at other addresses take longer to read: n 1024, 4 rows 4.4 (5.6), 8 rows 5.5 (5.8).
static bool few_rows(int dtype, const void *x, int64_t m, int64_t row_stride, int64_t n, int64_t k)
{
    const int64_t panels = (k + 255) / 256, size = dtype == TFTQ_F32 ? 4 : 2;
    const bool aligned = (uintptr_t)x % 16 == 0 && (m <= 1 || row_stride * size % 16 == 0);
    return m <= FEW_MOST && n <= FEW_WIDEST && FEW_SUMS + m * panels * FEW_PITCH <= 80 * 1024 && m * k * (1.0 + n / 4096.0) <= (aligned ? 1e5 : 4e4);
}

extern "C" int64_t tftq_mx_linear_workspace(int dtype, const void *x, int64_t m, int64_t row_stride, int64_t n, int64_t k)
{
    if (dtype != TFTQ_F32 && dtype != TFTQ_F16 && dtype != TFTQ_BF16) return TFTQ_E_DTYPE;
    if (m < 0 || n < 0 || k < 0 || m > MX_MOST || n > MX_MOST || k > MX_MOST) return TFTQ_E_SHAPE;
    return few_rows(dtype, x, m, row_stride, n, k) ? 0 : tftq_mx_bytes(m, k);
}

extern "C" int tftq_mx_linear(int dtype, const void *x, int64_t m, int64_t row_stride, const void *b, int64_t n, int64_t k,
                              void *out, int64_t out_stride, void *workspace, int64_t workspace_bytes, int device, void *stream)
{
    if (dtype != TFTQ_F32 && dtype != TFTQ_F16 && dtype != TFTQ_BF16) return TFTQ_E_DTYPE;
    if (m < 0 || n < 0 || k < 0 || m > MX_MOST || n > MX_MOST || k > MX_MOST) return TFTQ_E_SHAPE;
    if (m == 0 || n == 0) return 0;
    if (!out || out_stride < (m > 1 ? n : 0)) return TFTQ_E_ARG;
    if (k > 0 && (!x || !b || ((uintptr_t)b & 15) || row_stride < (m > 1 ? k : 0))) return TFTQ_E_ARG;
    if (k > 0 && few_rows(dtype, x, m, row_stride, n, k)) {
        DeviceScope scope(device);
        if (scope.err != hipSuccess) return (int)scope.err;
        const MxMatrix mb = mx_matrix((void *)b, n, k);
        const TileOperand tb = {mb.panels, mb.scales, (int)n};
        hipStream_t st = (hipStream_t)stream;
        switch (dtype) {
        case TFTQ_F32: return few<MxF32, TFTQ_F32>((const uint8_t *)x, row_stride, nullptr, (int)m, tb, (int)k, (uint8_t *)out, out_stride, st);
        case TFTQ_F16: return few<MxF16, TFTQ_F16>((const uint8_t *)x, row_stride, nullptr, (int)m, tb, (int)k, (uint8_t *)out, out_stride, st);
        default: return few<MxBF16, TFTQ_BF16>((const uint8_t *)x, row_stride, nullptr, (int)m, tb, (int)k, (uint8_t *)out, out_stride, st);
        }
    }
    if (k > 0) {
        if (workspace_bytes < tftq_mx_bytes(m, k)) return TFTQ_E_SIZE;
        if (!workspace) return TFTQ_E_ARG;
        if (const int rc = tftq_mx_quantize(dtype, x, m, k, row_stride, workspace, nullptr, device, stream)) return rc;
    }
    return tftq_mx_product(dtype, workspace, m, b, n, k, out, out_stride, device, stream);
}
