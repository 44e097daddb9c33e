// The product of two 4-bit microscaled matrices, c[i][j] = sum_k a[i][k] b[j][k], and its C entry.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tftq_device.h"
#include "tftq_mxfp4.h"

template <int DTYPE>
struct MxOut {
    static constexpr int SIZE = DTYPE == TFTQ_F32 ? 4 : 2, V = 16 / SIZE;
    __device__ static void put(uint8_t *to, float v)
    {
        if constexpr (DTYPE == TFTQ_F32) *(float *)to = v;
        else if constexpr (DTYPE == TFTQ_F16) *(_Float16 *)to = (_Float16)v;
        else *(__bf16 *)to = (__bf16)v;
    }
    __device__ static void put_vector(uint8_t *to, const float *v)
    {
        tile_i4 w;
        if constexpr (DTYPE == TFTQ_F32) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = __float_as_int(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint16_t lo = DTYPE == TFTQ_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) : __builtin_bit_cast(uint16_t, (__bf16)v[2 * i]);
                const uint16_t hi = DTYPE == TFTQ_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) : __builtin_bit_cast(uint16_t, (__bf16)v[2 * i + 1]);
                w[i] = (int)(lo | (uint32_t)hi << 16);
            }
        }
        *(tile_i4 *)to = w;
    }
};

template <class T, int DTYPE>
__global__ __launch_bounds__(T::THREADS) void k_mx_product(TileOperand a, TileOperand b, int panels, uint8_t *out, int64_t ld,
                                                           int whole, int tiles_m, int tiles_n)
{
    __shared__ __attribute__((aligned(128))) uint8_t lds[T::LDS];
    using O = MxOut<DTYPE>;
    int tm, tn;
    tile_place(tile_piece(blockIdx.x, gridDim.x), tiles_m, tiles_n, &tm, &tn);
    T t;
    t.zero();
    t.multiply(TilePair{a, b}, 0, panels, tm * T::ROWS, tn * T::COLS, lds);
    t.store_strips(tm * T::ROWS, tn * T::COLS, lds, [&](const float *strip, int row, int col) {
        const int lane = threadIdx.x & 63;
        if (whole) {
            constexpr int ACROSS = T::WN / O::V, AT_ONCE = 64 / ACROSS;
            const int c = lane % ACROSS * O::V;
            if (col + c >= b.rows) return;
#pragma unroll
            for (int r = lane / ACROSS; r < 32; r += AT_ONCE)
                if (row + r < a.rows) O::put_vector(out + ((int64_t)(row + r) * ld + col + c) * O::SIZE, strip + r * T::PITCH + c);
        } else {
            for (int r = 0; r < 32 && row + r < a.rows; r++)
                for (int c = lane; c < T::WN && col + c < b.rows; c += 64)
                    O::put(out + ((int64_t)(row + r) * ld + col + c) * O::SIZE, strip[r * T::PITCH + c]);
        }
    });
}

// A launch of tiles of one size.
template <class T>
static int product(int dtype, const TileOperand &a, const TileOperand &b, int panels, uint8_t *out, int64_t ld, hipStream_t st)
{
    const int size = dtype == TFTQ_F32 ? 4 : 2;
    int tiles_m = (a.rows + T::ROWS - 1) / T::ROWS, tiles_n = (b.rows + T::COLS - 1) / T::COLS;
    if ((int64_t)tiles_m * tiles_n > (1 << 22)) return TFTQ_E_SHAPE;
    int whole = ld * size % 16 == 0 && b.rows * size % 16 == 0 && (uintptr_t)out % 16 == 0;
    void *args[] = {(void *)&a, (void *)&b, (void *)&panels, (void *)&out, (void *)&ld, (void *)&whole, (void *)&tiles_m, (void *)&tiles_n};
    const void *k = dtype == TFTQ_F32 ? (const void *)k_mx_product<T, TFTQ_F32>
                    : dtype == TFTQ_F16 ? (const void *)k_mx_product<T, TFTQ_F16>
                                        : (const void *)k_mx_product<T, TFTQ_BF16>;
    return (int)hipLaunchKernel(k, dim3((unsigned)(tiles_m * tiles_n)), dim3(T::THREADS), args, 0, st);
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
    const int64_t big = ((m + 255) / 256) * ((n + 255) / 256), middle = ((m + 127) / 128) * ((n + 127) / 128);
    if (big >= 160) return product<Tile<256, 256, 2, 4, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    if (middle >= 160) return product<Tile<128, 128, 2, 2, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    return product<Tile<64, 64, 2, 2, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
}
