// What the kernels of row operators share (tftq_norm.hip, tftq_dropout.hip, tftq_embedding.hip, tftq_experts.hip).
//
// A row is a run of `cols` elements at any address that is a multiple of the element's size.  A team of
// lanes takes it in vectors of 16 bytes: lane l of the team has the vectors l, l + TEAM, l + 2 TEAM, ...
// The last vector may hold fewer elements; what lies past the row reads as zero and is not written.
#pragma once

#include "tftq_device.h"

typedef u32x4 u32x4_a1 __attribute__((aligned(1)));
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef u32 u32_a1 __attribute__((aligned(1)));
typedef uint16_t uint16_a1 __attribute__((aligned(1)));

// Rows of a launch: every team is whole, and a grid has fewer than 2^32 threads.
constexpr int64_t ROWS_THREADS = (int64_t)1 << 31;
constexpr int64_t ROWS_MOST = ((int64_t)1 << 31) - 65536;  // rows, columns, tokens and choices are at most so many

template <int ESZ> struct RowWord;
template <> struct RowWord<1> { typedef uint8_t type; };
template <> struct RowWord<2> { typedef uint16_t type; };
template <> struct RowWord<4> { typedef uint32_t type; };

// Elements col to col + 16 / ESZ - 1 of the row at `row` in two steps: fetch_row asks memory for them, settle_row puts
// them in their places.  The last vector of a row is fetched further ahead, so that it ends with the row, and
// moved down afterwards: no lane waits for memory before all it needs has been asked for (with the two in one, rows
// of 333 bf16 columns took 2.6 TB/s).  A row of fewer elements than a vector is fetched one by one.
template <int ESZ, bool STREAM = true>
DEV u32x4 fetch_row(uint64_t row, int col, int cols)
{
    constexpr int EPV = 16 / ESZ;
    typedef typename RowWord<ESZ>::type Word;
    u32x4 v = {0, 0, 0, 0};
    if (cols >= EPV) {
        if (col < cols) {
            const GLOBAL u32x4_a1 *at = as_global<const u32x4_a1>(row + (uint64_t)(u32)min(col, cols - EPV) * ESZ);
            if (STREAM) v = LOAD_STREAM(at);
            else v = *at;
        }
    } else if (col == 0) {
#pragma unroll
        for (int i = 0; i < EPV - 1; i++)
            if (i < cols) v[i * ESZ / 4] |= (u32)as_global<const Word>(row)[i] << (i * ESZ % 4 * 8);
    }
    return v;
}
template <int ESZ>
DEV u32x4 settle_row(u32x4 w, int col, int cols)
{
    constexpr int EPV = 16 / ESZ;
    const int over = col + EPV - cols;  // elements past the row
    if (cols >= EPV && over > 0 && over < EPV) {
        const u32 n = (u32)over * ESZ >> 2, sh = ((u32)over * ESZ & 3) * 8;
        const u32 a[5] = {n == 0 ? w.x : n == 1 ? w.y : n == 2 ? w.z : w.w, n == 0 ? w.y : n == 1 ? w.z : n == 2 ? w.w : 0u,
                          n == 0 ? w.z : n == 1 ? w.w : 0u, n == 0 ? w.w : 0u, 0u};
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = ESZ == 4 ? a[i] : (u32)((((uint64_t)a[i + 1] << 32) | a[i]) >> sh);
    }
    return w;
}
// Both at once, where nothing else is under way.
template <int ESZ, bool STREAM = true>
DEV u32x4 load_row(uint64_t row, int col, int cols) { return settle_row<ESZ>(fetch_row<ESZ, STREAM>(row, col, cols), col, cols); }

template <int ESZ, bool STREAM = true>
DEV void store_row(uint64_t row, int col, int cols, u32x4 v)
{
    constexpr int EPV = 16 / ESZ;
    uint64_t at = row + (uint64_t)(u32)col * ESZ;
    const int left = cols - col;
    if (left >= EPV) {
        if (STREAM) STORE_STREAM(v, as_global<u32x4_a1>(at));
        else *as_global<u32x4_a1>(at) = v;
    } else if (left > 0) {  // 8, 4, 2 and 1 bytes
        const u32 bytes = (u32)left * ESZ;
        if (bytes & 8) {
            *as_global<u32x2_a1>(at) = u32x2{v.x, v.y};
            v.x = v.z;
            v.y = v.w;
            at += 8;
        }
        if (bytes & 4) {
            *as_global<u32_a1>(at) = v.x;
            v.x = v.y;
            at += 4;
        }
        if (ESZ <= 2 && (bytes & 2)) {
            *as_global<uint16_a1>(at) = (uint16_t)v.x;
            v.x >>= 16;
            at += 2;
        }
        if (ESZ == 1 && (bytes & 1)) *as_global<uint8_t>(at) = (uint8_t)v.x;
    }
}

// The sum over the team's lanes, in an order that the team alone decides; every lane gets it.
// lds: TEAM / 64 floats for teams of several wavefronts, which are a whole workgroup.
template <int TEAM>
DEV float team_sum(float v, float *lds)
{
    if (TEAM >= 2) v += dpp_mov<0xB1>(v);
    if (TEAM >= 4) v += dpp_mov<0x4E>(v);
    if (TEAM >= 8) v += dpp_mov<0x141>(v);
    if (TEAM >= 16) v += dpp_mov<0x140>(v);
    if (TEAM >= 32) {
        const float a = bcast_lane(v, 0), b = bcast_lane(v, 16), c = bcast_lane(v, 32), d = bcast_lane(v, 48);
        if (TEAM == 32) v = (threadIdx.x & 32) ? c + d : a + b;
        else v = (a + b) + (c + d);
    }
    if (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < TEAM / 64; i++) v += lds[i];
        __syncthreads();
    }
    return v;
}
// Two sums at once; lds: twice as much.
template <int TEAM>
DEV void team_sum2(float &a, float &b, float *lds)
{
    if (TEAM <= 64) {
        a = team_sum<TEAM>(a, lds);
        b = team_sum<TEAM>(b, lds);
        return;
    }
    a = team_sum<64>(a, lds);
    b = team_sum<64>(b, lds);
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = a;
        lds[TEAM / 64 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < TEAM / 64; i++) {
        a += lds[i];
        b += lds[TEAM / 64 + i];
    }
    __syncthreads();
}
template <int TEAM>
DEV float team_largest(float v, float *lds)
{
    v = team_max<(TEAM > 64 ? 64 : TEAM)>(v, lds);
    if (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TEAM / 64; i++) v = fmaxf(v, lds[i]);
        __syncthreads();
    }
    return v;
}

// How many lanes take a row, and how many vectors each.
struct RowShape {
    int team, nv;
};

static inline bool rows_ok(int64_t rows, int64_t cols) { return rows >= 0 && cols >= 0 && rows <= ROWS_MOST && cols <= ROWS_MOST; }
static inline bool dtype_ok(int dtype) { return dtype == TFTQ_F32 || dtype == TFTQ_F16 || dtype == TFTQ_BF16; }
static inline int dtype_size(int dtype) { return dtype == TFTQ_F32 ? 4 : 2; }
