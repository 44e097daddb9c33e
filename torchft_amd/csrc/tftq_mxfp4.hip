// 4-bit microscaled matrices: quantisation along rows and columns, and the values back.
//
// Blocks of 32 consecutive elements of the contracted axis share a scale X = 2^e with
// e = clamp(floor(log2(max |x|)) - 2, -127, 127), held as the byte e + 127; every element is the nearest
// of 0, .5, 1, 1.5, 2, 3, 4, 6 to x / X with its sign, ties to the even mantissa, larger ones 6 (the
// OCP microscaling formats' E8M0 and E2M1).  A power of two divides exactly, so every step but the
// rounding to 4 bits is exact.  A block with an infinity or a NaN gets the byte 255, which is NaN.
//
// The matrix is kept in the panels that the product reads (tftq_tile.h): panel s holds 256 columns,
// 128 bytes of each row one after the other; then the scales, 8 bytes of each row and panel, with an
// even number of rows per panel.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tftq_mxfp4.h"

// The largest over the 32 / V neighbouring lanes that hold a row's block.
template <class T>
__device__ static inline uint32_t mx_over_block(uint32_t m)
{
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));   // lane ^ 1
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));   // lane ^ 2
    if (T::V == 4) m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));  // 7 - lane of 8
    return m;
}

// One wavefront per tile of 128 columns: a lane holds 16 bytes of P consecutive rows, so that a block
// of a column lies in one lane (P = 32) and a block of a row in 4 or 8 neighbouring ones: neither needs
// LDS, and the matrix is read once for both directions.  Bound by memory, and with both directions by the
// work between loads and stores: 14336x4096 bf16 along both axes 41 us (179 MB, 4.4 TB/s), 8192x4096 along
// rows 17 us (85 MB, 5.0 TB/s; a copy reaches 5.1).  P = 32 keeps 128 registers of data a lane: two
// wavefronts to a SIMD.
template <class T, bool BY_ROWS, bool BY_COLS, int P>
__global__ __launch_bounds__(64, 2) void k_mx_quantize(const uint8_t *x, int64_t ld, int rows, int cols, int tiles_c,
                                                       int row0, MxMatrix by_rows, MxMatrix by_cols)
{
    constexpr int V = T::V, ACROSS = 128 / V, GROUPS = 64 / ACROSS;
    static_assert(!BY_COLS || P == 32, "");
    const int piece = tile_piece(blockIdx.x, gridDim.x);
    const int lane = threadIdx.x;
    const int col = piece % tiles_c * 128 + lane % ACROSS * V;
    const int row = row0 + (piece / tiles_c * GROUPS + lane / ACROSS) * P;

    mx_u4 raw[P];
    const uint8_t *at = x + ((int64_t)row * ld + col) * T::SIZE;
    if (col + V <= cols) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            raw[p] = mx_u4{0, 0, 0, 0};
            if (row + p < rows) raw[p] = __builtin_nontemporal_load((const mx_u4_any *)(at + (int64_t)p * ld * T::SIZE));
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; p++) {
            raw[p] = mx_u4{0, 0, 0, 0};
            if (row + p < rows) raw[p] = mx_read<T>(at - (int64_t)col * T::SIZE + (int64_t)p * ld * T::SIZE, col, cols);
        }
    }

    if (BY_ROWS) {
        // of two rows the even lane stores its and its neighbour's codes of the first, the odd one those of
        // the second; of four rows every lane of a block's first four stores one's scale
        const int odd = lane & 1, mine = lane & 3, team = lane % (32 / V);
        uint8_t *codes = by_rows.panels + ((int64_t)(col >> 8) * rows + row + odd) * PANEL_BYTES + (col & 255 & ~(2 * V - 1)) / 2;
        uint8_t *scales = by_rows.scales + ((int64_t)(col >> 8) * ((rows + 1) & ~1) + row + mine) * 8 + (col & 255) / 32;
        uint32_t byte = 0;
#pragma unroll
        for (int p = 0; p < P; p += 2) {
            uint32_t c[2];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t m = T::mag(raw[p + q][0]);
#pragma unroll
                for (int w = 1; w < 4; w++) m = T::mag_max(m, T::mag(raw[p + q][w]));
                const uint32_t b = mx_byte(T::bits(mx_over_block<T>(T::mag_all(m))));
                c[q] = mx_codes<T>(raw[p + q], mx_scale(b));
                if ((p + q) % 4 == mine) byte = b;
            }
            const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? c[0] : c[1]), 0xb1, 0xf, 0xf, true);
            const uint32_t low = odd ? got : c[0], high = odd ? c[1] : got;
            if (row + p + odd < rows) {
                if (T::SIZE == 4) *(uint32_t *)(codes + p * PANEL_BYTES) = low | high << 16;
                else *(uint64_t *)(codes + p * PANEL_BYTES) = low | (uint64_t)high << 32;
            }
            if (p % 4 == 2 && team < 4 && row + p - 2 + mine < rows) scales[(p - 2) * 8] = (uint8_t)byte;
        }
    }
    if constexpr (BY_COLS) {
        uint8_t *codes = by_cols.panels + ((int64_t)(row >> 8) * cols + col) * PANEL_BYTES + (row & 255) / 2;
        uint8_t *scales = by_cols.scales + ((int64_t)(row >> 8) * ((cols + 1) & ~1) + col) * 8 + (row & 255) / 32;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            uint32_t m = T::mag(raw[0][w]);
#pragma unroll
            for (int p = 1; p < P; p++) m = T::mag_max(m, T::mag(raw[p][w]));
#pragma unroll
            for (int h = 0; h < 4 / T::SIZE; h++) {  // the word's columns
                const uint32_t byte = mx_byte(T::bits(T::SIZE == 4 ? m : h ? m >> 16 : m & 0xffffu));
                const float scale = mx_scale(byte);
                mx_u4 out;
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    uint32_t c = 0;
                    if constexpr (T::SIZE == 4) {
                        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(raw[8 * d][w]), __uint_as_float(raw[8 * d + 1][w]), scale, 0);
                        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(raw[8 * d + 2][w]), __uint_as_float(raw[8 * d + 3][w]), scale, 1);
                        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(raw[8 * d + 4][w]), __uint_as_float(raw[8 * d + 5][w]), scale, 2);
                        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(raw[8 * d + 6][w]), __uint_as_float(raw[8 * d + 7][w]), scale, 3);
                    } else {
                        const uint32_t pick = h ? 0x07060302u : 0x05040100u;  // the halves of two rows
                        c = T::template codes<0>(c, __builtin_amdgcn_perm(raw[8 * d + 1][w], raw[8 * d][w], pick), scale);
                        c = T::template codes<1>(c, __builtin_amdgcn_perm(raw[8 * d + 3][w], raw[8 * d + 2][w], pick), scale);
                        c = T::template codes<2>(c, __builtin_amdgcn_perm(raw[8 * d + 5][w], raw[8 * d + 4][w], pick), scale);
                        c = T::template codes<3>(c, __builtin_amdgcn_perm(raw[8 * d + 7][w], raw[8 * d + 6][w], pick), scale);
                    }
                    out[d] = c;
                }
                const int j = w * (4 / T::SIZE) + h;
                if (col + j < cols) {
                    *(mx_u4 *)(codes + j * PANEL_BYTES) = out;
                    scales[j * 8] = (uint8_t)byte;
                }
            }
        }
    }
}

// A lane turns V neighbouring codes into a vector of 16 bytes; codes are read in the order in which they lie.
// Bound by its stores: 14336x4096 to bf16 24 us (149 MB, 6.2 TB/s).
template <int DTYPE>
__global__ __launch_bounds__(256) void k_mx_dequantize(MxMatrix m, int rows, int cols, uint8_t *out, int64_t ld, int64_t first_group)
{
    constexpr int SIZE = DTYPE == TFTQ_F32 ? 4 : 2, V = 16 / SIZE, PER_ROW = 256 / V;
    const int64_t pieces = (int64_t)((cols + 255) >> 8) * rows * PER_ROW;
    const int64_t first = (first_group + blockIdx.x) * 1024 + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int64_t piece = first + 256 * q;
        if (piece >= pieces) return;
        const int64_t line = piece / PER_ROW;  // (panel, row)
        const int panel = (int)(line / rows), row = (int)(line - (int64_t)panel * rows), in = (int)(piece % PER_ROW);
        const int col = panel * 256 + in * V;
        if (col >= cols) continue;
        const uint32_t c = SIZE == 4 ? ((const uint16_t *)m.panels)[piece] : ((const uint32_t *)m.panels)[piece];
        const float scale = mx_scale(m.scales[((int64_t)panel * ((rows + 1) & ~1) + row) * 8 + in * V / 32]);
        const mx_f2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3)};
        mx_u4 w = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float v = (i & 1 ? p[i / 2].y : p[i / 2].x) * scale;
            if constexpr (DTYPE == TFTQ_F32) w[i] = __float_as_uint(v);
            else w[i / 2] |= (uint32_t)(DTYPE == TFTQ_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : __builtin_bit_cast(uint16_t, (__bf16)v)) << (16 * (i & 1));
        }
        uint8_t *to = out + ((int64_t)row * ld + col) * SIZE;
        if (col + V <= cols) {
            __builtin_nontemporal_store(w, (mx_u4_any *)to);
            continue;
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (col + i >= cols) continue;
            if (SIZE == 4) ((uint32_t *)to)[i] = w[i];
            else ((uint16_t *)to)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

static int64_t mx_panels(int64_t cols) { return (cols + 255) / 256; }

extern "C" int64_t tftq_mx_bytes(int64_t rows, int64_t cols)
{
    if (rows < 0 || cols < 0 || rows > MX_MOST || cols > MX_MOST) return TFTQ_E_SHAPE;
    return mx_panels(cols) * (rows * PANEL_BYTES + ((rows + 1) & ~(int64_t)1) * 8);
}

MxMatrix mx_matrix(void *buffer, int64_t rows, int64_t cols)
{
    return {(uint8_t *)buffer, buffer ? (uint8_t *)buffer + mx_panels(cols) * rows * PANEL_BYTES : nullptr};
}

template <class T>
static int quantize(const void *x, int64_t ld, int rows, int cols, const MxMatrix &r, const MxMatrix &c, hipStream_t st)
{
    constexpr int GROUPS = 64 / (128 / T::V);
    const int per_lane = c.panels ? 32 : 4;
    // every column of the last panel, and with columns every row of their last panel, is written
    int tc = (int)(mx_panels(cols) * 2);
    const int64_t high = c.panels ? mx_panels(rows) * 256 : rows, each = GROUPS * per_lane, tiles_r = (high + each - 1) / each;
    const uint8_t *px = (const uint8_t *)x;
    const void *k = !c.panels ? (const void *)k_mx_quantize<T, true, false, 4>
                    : r.panels ? (const void *)k_mx_quantize<T, true, true, 32>
                               : (const void *)k_mx_quantize<T, false, true, 32>;
    // 2^31 threads of a launch at most; a row has fewer than 2^24 tiles
    const int64_t at_once = (1 << 25) / tc;
    for (int64_t t = 0; t < tiles_r; t += at_once) {
        int row0 = (int)(t * each);
        void *args[] = {(void *)&px, (void *)&ld, (void *)&rows, (void *)&cols, (void *)&tc, (void *)&row0, (void *)&r, (void *)&c};
        const dim3 grid((unsigned)(std::min(at_once, tiles_r - t) * tc)), block(64);
        if (const int rc = (int)hipLaunchKernel(k, grid, block, args, 0, st)) return rc;
    }
    return 0;
}

extern "C" int tftq_mx_quantize(int dtype, const void *x, int64_t rows, int64_t cols, int64_t row_stride, void *by_rows,
                                void *by_cols, int device, void *stream)
{
    if (dtype != TFTQ_F32 && dtype != TFTQ_F16 && dtype != TFTQ_BF16) return TFTQ_E_DTYPE;
    if (rows < 0 || cols < 0 || rows > MX_MOST || cols > MX_MOST) return TFTQ_E_SHAPE;
    if (rows == 0 || cols == 0) return 0;
    if (!by_rows && !by_cols) return TFTQ_E_ARG;
    if (((uintptr_t)by_rows | (uintptr_t)by_cols) & 15) return TFTQ_E_ARG;
    if (!x || row_stride < (rows > 1 ? cols : 0)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const MxMatrix r = mx_matrix(by_rows, rows, cols), c = mx_matrix(by_cols, cols, rows);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case TFTQ_F32: return quantize<MxF32>(x, row_stride, (int)rows, (int)cols, r, c, st);
    case TFTQ_F16: return quantize<MxF16>(x, row_stride, (int)rows, (int)cols, r, c, st);
    default: return quantize<MxBF16>(x, row_stride, (int)rows, (int)cols, r, c, st);
    }
}

extern "C" int tftq_mx_dequantize(int dtype, const void *matrix, int64_t rows, int64_t cols, void *out, int64_t row_stride,
                                  int device, void *stream)
{
    if (dtype != TFTQ_F32 && dtype != TFTQ_F16 && dtype != TFTQ_BF16) return TFTQ_E_DTYPE;
    if (rows < 0 || cols < 0 || rows > MX_MOST || cols > MX_MOST) return TFTQ_E_SHAPE;
    if (rows == 0 || cols == 0) return 0;
    if (!matrix || !out || ((uintptr_t)matrix & 15) || row_stride < (rows > 1 ? cols : 0)) return TFTQ_E_ARG;
    const int64_t groups = (mx_panels(cols) * rows * (dtype == TFTQ_F32 ? 64 : 32) + 1023) / 1024;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    MxMatrix m = mx_matrix((void *)matrix, rows, cols);
    int r = (int)rows, c = (int)cols;
    constexpr int64_t AT_ONCE = 1 << 23;  // 2^31 threads
    int64_t first = 0;
    void *args[] = {(void *)&m, (void *)&r, (void *)&c, (void *)&out, (void *)&row_stride, (void *)&first};
    const void *k = dtype == TFTQ_F32 ? (const void *)k_mx_dequantize<TFTQ_F32>
                    : dtype == TFTQ_F16 ? (const void *)k_mx_dequantize<TFTQ_F16>
                                        : (const void *)k_mx_dequantize<TFTQ_BF16>;
    for (; first < groups; first += AT_ONCE)
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)std::min(AT_ONCE, groups - first)), dim3(256), args, 0, (hipStream_t)stream))
            return rc;
    return 0;
}
