// Dropout from a counter-based generator: out = residual + x keep / (1 - p), and the same of a gradient.
//
// Random numbers are those of Philox with four 32-bit words and ten rounds (J. Salmon et al., "Parallel random
// numbers: as easy as 1, 2, 3", 2011), its key the seed, its counter the number of a block of eight elements and
// the caller's offset: a word is two numbers of 16 bits, and an element stays if its number is at least
// round(p 65536).  So the mask is a function of seed, offset and place, is never stored, and is the same for any
// launch.  16 bits an element halve the rounds: with a call for four elements the multiplications of 32 bits,
// a quarter as fast as others, take longer than memory does; p is a multiple of 2^-16 then.
#include "tftq_rows.h"

struct DropoutArgs {
    uint64_t x, residual, out, seed_at;  // residual, seed_at: 0 for none
    uint64_t seed, offset;
    int64_t n, first;  // elements; the launch's first block of eight
    u32 threshold;
    float factor;
};

DEV u32x4 philox(u32x4 c, u32 k0, u32 k1)
{
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t p0 = (uint64_t)c.x * 0xD2511F53u, p1 = (uint64_t)c.z * 0xCD9E8D57u;
        c = u32x4{(u32)(p1 >> 32) ^ c.y ^ k0, (u32)p1, (u32)(p0 >> 32) ^ c.w ^ k1, (u32)p0};
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

// A lane takes two blocks of eight elements; the last one may be shorter.  Bound by memory: 8192x4096 bf16 onto a residual
// 33 us (201 MB, 6.1 TB/s), without 22 (134 MB, 6.1).
template <class T>
__global__ __launch_bounds__(256) void k_dropout(const DropoutArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, NV = 8 / EPV, U = 2;
    const uint64_t seed = a.seed_at ? *as_global<const uint64_t>(a.seed_at) : a.seed;
    u32x4 raw[U][NV], res[U][NV];
    int left[U];  // bytes
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t block = a.first + (int64_t)blockIdx.x * (256 * U) + u * 256 + threadIdx.x, rest = a.n - block * 8;
        left[u] = rest < 0 ? 0 : rest > 8 ? 8 * ESZ : (int)rest * ESZ;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const uint64_t at = (uint64_t)(block * 8) * ESZ + v * 16;
            const bool whole = left[u] >= (v + 1) * 16;
            raw[u][v] = res[u][v] = u32x4{0, 0, 0, 0};
            if (whole) {
                raw[u][v] = LOAD_STREAM(as_global<const u32x4_a1>(a.x + at));
                if (a.residual) res[u][v] = LOAD_STREAM(as_global<const u32x4_a1>(a.residual + at));
            } else if (left[u] > v * 16) {
                raw[u][v] = load_bytes(a.x + at, (u32)(left[u] - v * 16));
                if (a.residual) res[u][v] = load_bytes(a.residual + at, (u32)(left[u] - v * 16));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t block = a.first + (int64_t)blockIdx.x * (256 * U) + u * 256 + threadIdx.x;
        const u32x4 words = philox(u32x4{(u32)block, (u32)((uint64_t)block >> 32), (u32)a.offset, (u32)(a.offset >> 32)}, (u32)seed, (u32)(seed >> 32));
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float f[EPV], r[EPV];
            Elem<T>::unpack(raw[u][v], f);
            Elem<T>::unpack(res[u][v], r);
#pragma unroll
            for (int i = 0; i < EPV; i++) {
                const int e = v * EPV + i;
                const u32 number = e & 1 ? words[e / 2] >> 16 : words[e / 2] & 0xFFFFu;
                f[i] = number >= a.threshold ? f[i] * a.factor : 0.0f;
                if (a.residual) f[i] += r[i];
            }
            const uint64_t to = a.out + (uint64_t)(block * 8) * ESZ + v * 16;
            const u32x4 out = Elem<T>::pack(f);
            if (left[u] >= (v + 1) * 16) STORE_STREAM(out, as_global<u32x4_a1>(to));
            else if (left[u] > v * 16) store_bytes(to, (u32)(left[u] - v * 16), out);
        }
    }
}

extern "C" int tftq_dropout(int dtype, const void *x, const void *residual, int64_t n, double p, int64_t seed, const int64_t *seed_at,
                            int64_t offset, void *out, int device, void *stream)
{
    if (!dtype_ok(dtype)) return TFTQ_E_DTYPE;
    if (n < 0) return TFTQ_E_SHAPE;
    if (!(p >= 0.0 && p <= 1.0)) return TFTQ_E_ARG;
    if (n == 0) return 0;
    if (!x || !out || ((uintptr_t)seed_at & 7)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const u32 threshold = (u32)__builtin_rint(p * 65536.0);
    DropoutArgs a = {(uint64_t)x, (uint64_t)residual, (uint64_t)out, (uint64_t)seed_at, (uint64_t)seed, (uint64_t)offset, n, 0,
                     threshold, threshold < 65536 ? (float)(65536.0 / (65536.0 - threshold)) : 0.0f};
    const void *k = dtype == TFTQ_F32 ? (const void *)k_dropout<float> : dtype == TFTQ_F16 ? (const void *)k_dropout<f16_tag> : (const void *)k_dropout<bf16_tag>;
    const int64_t blocks = (n + 7) / 8, at_once = ROWS_THREADS;
    for (; a.first < blocks; a.first += at_once) {
        void *args[] = {(void *)&a};
        const int64_t now = std::min(at_once, blocks - a.first);
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)((now + 511) / 512)), dim3(256), args, 0, (hipStream_t)stream)) return rc;
    }
    return 0;
}
