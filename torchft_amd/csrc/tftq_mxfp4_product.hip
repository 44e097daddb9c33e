// The product of two 4-bit microscaled matrices, c[i][j] = sum_k a[i][k] b[j][k], and its C entry.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tftq_device.h"
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
};

template <class T, int DTYPE>
__global__ __launch_bounds__(T::THREADS) void k_mx_product(TileOperand a, TileOperand b, int panels, uint8_t *out, int64_t ld,
                                                           int whole, int tiles_m, int tiles_n)
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
        t.template store_pieces<O::SIZE>(row0, col0, lds + 2 * T::BUFFER, O::two, [&](tile_i4 v, int row, int col) {
            if (row >= a.rows) return;
            uint8_t *at = out + ((int64_t)row * ld + col) * O::SIZE;
            if (whole) {
                if (col < b.rows) *(tile_i4 *)at = v;
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
    const int64_t big = ((m + 255) / 256) * ((n + 255) / 256), middle = ((m + 127) / 128) * ((n + 127) / 128);
    if (big >= 160) return product<Tile<256, 256, 2, 4, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    if (middle >= 160) return product<Tile<128, 128, 2, 2, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
    return product<Tile<64, 64, 2, 2, true>>(dtype, ta, tb, panels, (uint8_t *)out, row_stride, st);
}
