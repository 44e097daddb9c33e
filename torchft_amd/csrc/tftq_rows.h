// What the kernels of row operators share (tftq_norm.hip, tftq_dropout.hip, tftq_embedding.hip, tftq_experts.hip).
//
// A row is a run of `cols` elements at any address that is a multiple of the element's size.  A team of
// lanes takes it in vectors of 16 bytes: lane l of the team has the vectors l, l + TEAM, l + 2 TEAM, ...  Where a row is
// no whole number of vectors its last one is moved back to end with the row: the elements that two lanes
// then have (Piece::over of the later one) are the same in both, are stored twice, and count in a sum once.  So every load and
// store is a whole vector and no lane waits for one before it has asked for all (rows of 333 bf16 columns whose last
// vector was read element by element took 2.6 TB/s, now 5).  Rows shorter than a vector have kernels of their own (NARROW), where the first
// lane has all of the row and zeros behind it.
#pragma once

#include "tftq_device.h"

typedef u32x4 u32x4_a1 __attribute__((aligned(1)));
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef u32 u32_a1 __attribute__((aligned(1)));
typedef uint16_t uint16_a1 __attribute__((aligned(1)));

// Rows of a launch: every team is whole, and a grid has fewer than 2^32 threads.
constexpr int64_t ROWS_THREADS = (int64_t)1 << 31;
constexpr int64_t ROWS_MOST = ((int64_t)1 << 31) - 65536;  // rows, columns, tokens and choices are at most so many

// The first n (0 to 16) bytes at an address, zeros behind, and back.
DEV u32x4 load_bytes(uint64_t at, u32 n)
{
    if (n >= 16) return *as_global<const u32x4_a1>(at);
    u32x4 v = {0, 0, 0, 0};
    u32 low = 0, high = 0;
    if (n & 8) {
        const u32x2 w = *as_global<const u32x2_a1>(at);
        v.x = w.x;
        v.y = w.y;
        at += 8;
    }
    if (n & 4) {
        low = *as_global<const u32_a1>(at);
        at += 4;
    }
    if (n & 2) {
        high = *as_global<const uint16_a1>(at);
        at += 2;
    }
    if (n & 1) high |= (u32)*as_global<const uint8_t>(at) << (n & 2 ? 16 : 0);
    if (!(n & 4)) {
        low = high;
        high = 0;
    }
    if (n & 8) return u32x4{v.x, v.y, low, high};
    return u32x4{low, high, 0, 0};
}
DEV void store_bytes(uint64_t at, u32 n, u32x4 v)
{
    if (n >= 16) {
        *as_global<u32x4_a1>(at) = v;
        return;
    }
    if (n & 8) {
        *as_global<u32x2_a1>(at) = u32x2{v.x, v.y};
        v.x = v.z;
        v.y = v.w;
        at += 8;
    }
    if (n & 4) {
        *as_global<u32_a1>(at) = v.x;
        v.x = v.y;
        at += 4;
    }
    if (n & 2) {
        *as_global<uint16_a1>(at) = (uint16_t)v.x;
        v.x >>= 16;
        at += 2;
    }
    if (n & 1) *as_global<uint8_t>(at) = (uint8_t)v.x;
}

// Where a lane's vector of EPV elements is in a row, for the column at which it would begin if it were not moved.
struct Piece {
    bool in;   // there is one
    int at;    // its first column
    int over;  // so many of its first elements belong to the lane before
};
template <int EPV, bool NARROW>
DEV Piece piece_of(int col, int cols)
{
    const int at = NARROW ? 0 : min(col, cols - EPV);
    return {NARROW ? col == 0 : col < cols, at, col - at};
}

// The vector at a piece, zeros where there is none, and back.
template <int ESZ, bool NARROW, bool STREAM = true>
DEV u32x4 load_row(uint64_t row, const Piece &p, int cols)
{
    u32x4 v = {0, 0, 0, 0};
    if (p.in) {
        const uint64_t at = row + (uint64_t)(u32)p.at * ESZ;
        if (NARROW) v = load_bytes(at, (u32)cols * ESZ);
        else if (STREAM) v = LOAD_STREAM(as_global<const u32x4_a1>(at));
        else v = *as_global<const u32x4_a1>(at);
    }
    return v;
}
template <int ESZ, bool NARROW, bool STREAM = true>
DEV void store_row(uint64_t row, const Piece &p, int cols, u32x4 v)
{
    if (!p.in) return;
    const uint64_t at = row + (uint64_t)(u32)p.at * ESZ;
    if (NARROW) store_bytes(at, (u32)cols * ESZ, v);
    else if (STREAM) STORE_STREAM(v, as_global<u32x4_a1>(at));
    else *as_global<u32x4_a1>(at) = v;
}

// Zeros for the elements that the lane before has too: before a sum over the row.
template <int EPV>
DEV void count_once(float (&f)[EPV], const Piece &p)
{
    if (p.over > 0) {
#pragma unroll
        for (int i = 0; i < EPV - 1; i++)
            if (i < p.over) f[i] = 0.0f;
    }
}

// fp32 sums of a row's columns, kept apart: EPV of them from a piece's first column on.  Their rows are
// sums_stride(cols) long, so that a narrow row has room for a vector.
static TFTQ_HD inline int64_t sums_stride(int64_t cols) { return cols < 8 ? 8 : (cols + 3) & ~(int64_t)3; }
template <int EPV>
DEV void store_sums(uint64_t row, const Piece &p, const float (&f)[EPV])
{
    if (!p.in) return;
#pragma unroll
    for (int i = 0; i < EPV; i += 4)
        *as_global<u32x4_a4>(row + (uint64_t)(u32)(p.at + i) * 4) = u32x4{as_u(f[i]), as_u(f[i + 1]), as_u(f[i + 2]), as_u(f[i + 3])};
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
