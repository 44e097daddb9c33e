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
// LDS, and the matrix is read once for both directions.
template <class T, bool BY_ROWS, bool BY_COLS, int P>
__global__ __launch_bounds__(64, 2) void k_mx_quantize(const uint8_t *x, int64_t ld, int rows, int cols, int tiles_c,
                                                       MxMatrix by_rows, MxMatrix by_cols)
{
    constexpr int V = T::V, ACROSS = 128 / V, GROUPS = 64 / ACROSS;
    static_assert(!BY_COLS || P == 32, "");
    const int piece = tile_piece(blockIdx.x, gridDim.x);
    const int lane = threadIdx.x;
    const int col = piece % tiles_c * 128 + lane % ACROSS * V;
    const int row = (piece / tiles_c * GROUPS + lane / ACROSS) * P;

    mx_u4 raw[P];
    const uint8_t *at = x + ((int64_t)row * ld + col) * T::SIZE;
    if (col + V <= cols) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            raw[p] = mx_u4{0, 0, 0, 0};
            if (row + p < rows) raw[p] = *(const mx_u4_any *)(at + (int64_t)p * ld * T::SIZE);
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; p++) {
            raw[p] = mx_u4{0, 0, 0, 0};
            if (row + p < rows) raw[p] = mx_read<T>(at - (int64_t)col * T::SIZE + (int64_t)p * ld * T::SIZE, col, cols);
        }
    }

    if (BY_ROWS) {
        uint8_t *codes = by_rows.panels + ((int64_t)(col >> 8) * rows + row) * PANEL_BYTES + (col & 255) / 2;
        uint8_t *scales = by_rows.scales + ((int64_t)(col >> 8) * ((rows + 1) & ~1) + row) * 8 + (col & 255) / 32;
#pragma unroll
        for (int p = 0; p < P; p++) {
            uint32_t m = T::mag(raw[p][0]);
#pragma unroll
            for (int w = 1; w < 4; w++) m = T::mag_max(m, T::mag(raw[p][w]));
            const uint32_t byte = mx_byte(T::bits(mx_over_block<T>(T::mag_all(m))));
            const float scale = mx_scale(byte);
            const uint32_t c = mx_codes<T>(raw[p], scale);
            if (row + p < rows) {
                if (T::SIZE == 4) *(uint16_t *)(codes + p * PANEL_BYTES) = (uint16_t)c;
                else *(uint32_t *)(codes + p * PANEL_BYTES) = c;
                if (lane % (32 / V) == 0) scales[p * 8] = (uint8_t)byte;
            }
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

template <int DTYPE>
__device__ static inline void mx_store(uint8_t *to, const float *v, int n, bool whole)
{
    if constexpr (DTYPE == TFTQ_F32) {
        if (whole) {
            ((float4 *)to)[0] = float4{v[0], v[1], v[2], v[3]};
            ((float4 *)to)[1] = float4{v[4], v[5], v[6], v[7]};
        } else {
            for (int i = 0; i < 8; i++)
                if (i < n) ((float *)to)[i] = v[i];
        }
    } else {
        uint16_t h[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            h[i] = DTYPE == TFTQ_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[i]) : __builtin_bit_cast(uint16_t, (__bf16)v[i]);
        if (whole) {
            mx_u4 w;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
            *(mx_u4 *)to = w;
        } else {
            for (int i = 0; i < 8; i++)
                if (i < n) ((uint16_t *)to)[i] = h[i];
        }
    }
}

// A lane turns 8 codes, a word of the panels, into 8 neighbouring elements; words are read in the
// order in which they lie.
template <int DTYPE>
__global__ __launch_bounds__(256) void k_mx_dequantize(MxMatrix m, int rows, int cols, uint8_t *out, int64_t ld, int whole)
{
    constexpr int SIZE = DTYPE == TFTQ_F32 ? 4 : 2;
    const int64_t words = (int64_t)((cols + 255) >> 8) * rows * 32;
    const int64_t first = (int64_t)blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int64_t word = first + 256 * q;
        if (word >= words) return;
        const int64_t line = word >> 5;  // (panel, row)
        const int panel = (int)(line / rows), row = (int)(line - (int64_t)panel * rows), in = (int)word & 31;
        const int col = panel * 256 + in * 8;
        if (col >= cols) continue;
        const uint32_t c = ((const uint32_t *)m.panels)[word];
        const float scale = mx_scale(m.scales[((int64_t)panel * ((rows + 1) & ~1) + row) * 8 + in / 4]);
        const mx_f2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3)};
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = p[i].x * scale, v[2 * i + 1] = p[i].y * scale;
        mx_store<DTYPE>(out + ((int64_t)row * ld + col) * SIZE, v, cols - col, whole && col + 8 <= cols);
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
    const int64_t tiles_c = mx_panels(cols) * 2;
    const int64_t high = c.panels ? mx_panels(rows) * 256 : rows;
    const int64_t tiles = tiles_c * ((high + GROUPS * per_lane - 1) / (GROUPS * per_lane));
    if (tiles > (1 << 25)) return TFTQ_E_SHAPE;
    const dim3 grid((unsigned)tiles), block(64);
    const uint8_t *px = (const uint8_t *)x;
    int tc = (int)tiles_c;
    void *args[] = {(void *)&px, (void *)&ld, (void *)&rows, (void *)&cols, (void *)&tc, (void *)&r, (void *)&c};
    const void *k = !c.panels ? (const void *)k_mx_quantize<T, true, false, 4>
                    : r.panels ? (const void *)k_mx_quantize<T, true, true, 32>
                               : (const void *)k_mx_quantize<T, false, true, 32>;
    return (int)hipLaunchKernel(k, grid, block, args, 0, st);
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
    const int64_t groups = (mx_panels(cols) * rows * 32 + 1023) / 1024;
    if (groups > (1 << 23)) return TFTQ_E_SHAPE;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    MxMatrix m = mx_matrix((void *)matrix, rows, cols);
    const int size = dtype == TFTQ_F32 ? 4 : 2;
    int whole = row_stride * size % 16 == 0 && (uintptr_t)out % 16 == 0, r = (int)rows, c = (int)cols;
    void *args[] = {(void *)&m, (void *)&r, (void *)&c, (void *)&out, (void *)&row_stride, (void *)&whole};
    const void *k = dtype == TFTQ_F32 ? (const void *)k_mx_dequantize<TFTQ_F32>
                    : dtype == TFTQ_F16 ? (const void *)k_mx_dequantize<TFTQ_F16>
                                        : (const void *)k_mx_dequantize<TFTQ_BF16>;
    return (int)hipLaunchKernel(k, dim3((unsigned)groups), dim3(256), args, 0, (hipStream_t)stream);
}
