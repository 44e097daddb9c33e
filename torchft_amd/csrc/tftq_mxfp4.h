// A 4-bit microscaled matrix in device memory, and what makes the codes and scales of numbers: shared by
// the quantisation and the product.
#pragma once

#include "tftq_device.h"
#include "tftq_tile.h"

constexpr int64_t MX_MOST = (1ll << 31) - 1024;  // rows or columns

struct MxMatrix {
    uint8_t *panels;
    uint8_t *scales;
};

// The parts of a buffer of tftq_mx_bytes(rows, cols) bytes; two null pointers for none.
__attribute__((visibility("hidden"))) MxMatrix mx_matrix(void *buffer, int64_t rows, int64_t cols);

typedef uint32_t mx_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_u4_any __attribute__((ext_vector_type(4), aligned(2)));  // at any element's address
typedef uint16_t mx_s2 __attribute__((ext_vector_type(2)));
typedef _Float16 mx_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_b2 __attribute__((ext_vector_type(2)));
typedef float mx_f2 __attribute__((ext_vector_type(2)));

// What the kernels ask of an element type: a 16-byte vector holds V elements in four words.  Magnitudes
// are compared as the integers that their bits are, two of a 16-bit type at once; an infinity or NaN is
// then larger than every finite value.
struct MxF32 {
    static constexpr int SIZE = 4, V = 4;
    __device__ static uint32_t mag(uint32_t w) { return w & 0x7fffffffu; }
    __device__ static uint32_t mag_max(uint32_t a, uint32_t b) { return max(a, b); }
    __device__ static uint32_t mag_all(uint32_t m) { return m; }  // the larger of a word's magnitudes
    __device__ static uint32_t bits(uint32_t m) { return m; }     // of a magnitude: its binary32 bits
};
struct MxHalf {
    static constexpr int SIZE = 2, V = 8;
    __device__ static uint32_t mag(uint32_t w) { return w & 0x7fff7fffu; }
    __device__ static uint32_t mag_max(uint32_t a, uint32_t b)
    {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(mx_s2, a), __builtin_bit_cast(mx_s2, b)));
    }
    __device__ static uint32_t mag_all(uint32_t m) { return max(m & 0xffffu, m >> 16); }
};
struct MxF16 : MxHalf {
    __device__ static uint32_t bits(uint32_t m) { return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m)); }
    template <int SEL>
    __device__ static uint32_t codes(uint32_t old, uint32_t w, float x)
    {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(mx_h2, w), x, SEL);
    }
};
struct MxBF16 : MxHalf {
    __device__ static uint32_t bits(uint32_t m) { return m << 16; }
    template <int SEL>
    __device__ static uint32_t codes(uint32_t old, uint32_t w, float x)
    {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(mx_b2, w), x, SEL);
    }
};

// The scale's byte for a block whose largest magnitude has these binary32 bits.  Subnormal numbers
// (exponent field 0) are below 2^-126, so their blocks have the smallest scale whatever they hold.
__device__ static inline uint32_t mx_byte(uint32_t bits)
{
    const int e = (int)(bits >> 23);
    return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// 2^(byte - 127) in binary32; 2^-127 is subnormal, and 255 is NaN.
__device__ static inline float mx_scale(uint32_t byte)
{
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

// The codes of the elements of a 16-byte vector, V / 2 bytes in the low end of the word.
template <class T>
__device__ static inline uint32_t mx_codes(mx_u4 w, float scale)
{
    uint32_t c = 0;
    if constexpr (T::SIZE == 4) {
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(w[0]), __uint_as_float(w[1]), scale, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(w[2]), __uint_as_float(w[3]), scale, 1);
    } else {
        c = T::template codes<0>(c, w[0], scale);
        c = T::template codes<1>(c, w[1], scale);
        c = T::template codes<2>(c, w[2], scale);
        c = T::template codes<3>(c, w[3], scale);
    }
    return c;
}
// Columns `col` to col + V - 1 of a row of which `cols` exist, the others zero.
template <class T>
__device__ static inline mx_u4 mx_read(const uint8_t *row, int col, int cols)
{
    const uint8_t *from = row + (int64_t)col * T::SIZE;
    if (col + T::V <= cols) return *(const mx_u4_any *)from;
    mx_u4 w = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < T::V; v++) {
        if (col + v >= cols) continue;
        if (T::SIZE == 4) w[v] = ((const uint32_t *)from)[v];
        else w[v / 2] |= (uint32_t)((const uint16_t *)from)[v] << (16 * (v & 1));
    }
    return w;
}
