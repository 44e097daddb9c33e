// Root-mean-square norm of rows, behind the residual's addition, and its gradients.
//
//    h = x + residual (rounded to the rows' type, and kept);  y = h r w,  r = 1 / sqrt(mean(h^2) + eps)
//    dx = r (g - h r^2 mean(g h)) + dh with g = dy w;  dw = sum over rows of dy h r
//
// Sums are fp32.  h is rounded before the norm, so that the gradients, which have nothing but the h that
// was kept, are those of the y that was returned; y is rounded once.  r is computed again in the backward
// pass: its sum of squares rides along with that of g h.
//
// y may leave in 8 bits: e4m3 codes with one fp32 scale a row, max |y| / 448, that multiplies them (1 where that
// is no normal number).  A code is the nearest to y / scale = 448 h w / max |h w|, in which r cancels, an even one where two are as
// near.  In fp32 that quotient is off by 5 2^-24 at most, so that the codes on both sides of it, 2^-21 away, differ once
// in 10^5 elements; there products in 64 bits, which are exact, say on which side of the border it lies, or on it.  Of bf16 rows and
// weights one in 2000 lies on a border; their products are exact in fp32 already.  8192x2048 fp32 25 us (26 with 64-bit products of all
// elements), 8192x4096 bf16 with a residual 40.2 (39.8 from an fp32 y, which had a quarter of the quotients on a border on the wrong side; 40.7
// with fp32 weights, 42.7 where these are ones: one in 130 is on a border).
#include "tftq_rows.h"

struct NormArgs {
    uint64_t x, residual, weight, y, h, codes, scales;  // residual, weight, h: 0 for none; codes and scales for 8 bits, else y
    int64_t x_stride, residual_stride;                  // bytes from row to row; all others are contiguous
    int64_t x_group_stride;                             // and from group to group of
    u32 x_group;                                        // so many rows of x
    int64_t row0, rows;
    int cols;
    float eps, inv_cols;
};

// Where a row begins among rows in groups.
DEV uint64_t row_at(uint64_t base, int64_t row, int64_t stride, u32 group, int64_t group_stride, int64_t rows)
{
    if (group >= rows) return base + (uint64_t)(row * stride);
    return base + (uint64_t)((int64_t)((u32)row / group) * group_stride + (int64_t)((u32)row % group) * stride);
}

// The weight's elements that belong to a vector: loaded early, widened late.  WIDE: the weight is fp32 and the rows are not.
template <class T, bool NARROW, bool WIDE>
struct Weights {
    static_assert(!WIDE || Elem<T>::EPV == 8, "");
    u32x4 raw[WIDE ? 2 : 1];
    DEV void load(uint64_t weight, const Piece &p, int cols)
    {
#pragma unroll
        for (int i = 0; i < (WIDE ? 2 : 1); i++) raw[i] = u32x4{0, 0, 0, 0};
        if (!weight || !p.in) return;
        if constexpr (!WIDE) raw[0] = load_row<Elem<T>::ESZ, NARROW, false>(weight, p, cols);
        else {
            const uint64_t at = weight + (uint64_t)(u32)p.at * 4;
            if (NARROW) {
                raw[0] = load_bytes(at, min(16u, (u32)cols * 4));
                if (cols > 4) raw[1] = load_bytes(at + 16, (u32)(cols - 4) * 4);
            } else {
                raw[0] = *as_global<const u32x4_a4>(at);
                raw[1] = *as_global<const u32x4_a4>(at + 16);
            }
        }
    }
    DEV void unpack(uint64_t weight, float (&w)[Elem<T>::EPV]) const
    {
        constexpr int EPV = Elem<T>::EPV;
        if (!weight) {
#pragma unroll
            for (int i = 0; i < EPV; i++) w[i] = 1.0f;
        } else if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < EPV; i++) w[i] = as_f(raw[i / 4][i % 4]);
        } else Elem<T>::unpack(raw[0], w);
    }
};

DEV float inverse_root(float mean_square, float eps) { return 1.0f / __builtin_sqrtf(mean_square + eps); }

// r as a power of two, by which h can be multiplied without rounding and without a product h w that passes fp32's range, and
// the rest, 1 or more and below 2.  NaN stays.
DEV void split_root(float r, float &unit, float &rest)
{
    unit = r != r ? r : as_f(as_u(r) & 0x7f800000u);
    rest = as_f((as_u(r) & 0x007fffffu) | 0x3f800000u);
}
// The largest |h unit w| of a row in 64 bits: `mine` is a lane's, rounded; where that is the row's, and not 0, left(mine) is the largest part that
// such numbers' rounding left out.  lds: 2 TEAM / 64 floats.
template <int TEAM, class F>
DEV double team_largest_product(float mine, float *lds, F left)
{
    constexpr int WAVES = TEAM / 64;
    constexpr float NONE = -__builtin_inff();
    float high = team_max<(TEAM > 64 ? 64 : TEAM)>(mine, lds), low = NONE;
    if (TEAM <= 64) {
        if (mine == high && high > 0.0f) low = left(high);
        low = team_max<(TEAM > 64 ? 64 : TEAM)>(low, lds);
    } else {
        const float wave = high;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = wave;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; i++) high = fmaxf(high, lds[i]);
        if (wave == high) {
            if (mine == high && high > 0.0f) low = left(high);
            low = team_max<64>(low, lds);
        }
        if ((threadIdx.x & 63) == 0) lds[WAVES + (threadIdx.x >> 6)] = low;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; i++) low = fmaxf(low, lds[WAVES + i]);
    }
    return (double)high + (high > 0.0f && high < __builtin_inff() ? low : 0.0f);
}

DEV float row_scale(float part, bool &normal)
{
    normal = part >= 0x1p-126f;
    return normal ? part : 1.0f;
}
// What a row's scale and codes are made with, from its largest |h unit w| and what that leaves of r.  Where the scale is 1 for want of a
// normal number all codes are zeros, or NaN.
struct RowCodes {
    float scale, under, over;
    double most;
    DEV RowCodes(double largest, float rest) : most(largest)
    {
        const float high = (float)largest;
        bool normal;
        scale = row_scale(high / 448.0f * rest, normal);
        const float by = normal ? 448.0f / high : 0.0f;
        under = by * 0x1.fffffp-1f;
        over = by * 0x1.000008p+0f;
    }
    // Of any products p = h unit w, rounded: the codes 2^-21 below and above 448 p / most, off by 5 2^-24 at most.  Where they differ,
    // the sign of 896 h unit w - (both codes' numbers) most, two products of 53 bits at most, says which it is.  wide(i): h unit w in 64 bits.
    template <int EPV, class F>
    DEV u32x2 codes(const float (&p)[EPV], F wide) const
    {
        u32 c[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < EPV; i += 4) {
            u32 code = pack_fp8x4(p[i] * under, p[i + 1] * under, p[i + 2] * under, p[i + 3] * under);
            const u32 differ = code ^ pack_fp8x4(p[i] * over, p[i + 1] * over, p[i + 2] * over, p[i + 3] * over);
            if (differ) {
                float lower[4], upper[4];
                unpack_fp8x4(code, lower);
                unpack_fp8x4(code ^ differ, upper);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const u32 mine = differ & 0xFFu << (8 * j);
                    if (!mine) continue;
                    const double above = __builtin_fma(-(double)__builtin_fabsf(lower[j] + upper[j]), most, 896.0 * __builtin_fabs(wide(i + j)));
                    if (above > 0.0 || (above == 0.0 && (code >> (8 * j) & 1))) code ^= mine;
                }
            }
            c[i / 4] = code;
        }
        return u32x2{c[0], c[1]};
    }
};
// Of products n = 7/8 h unit w that are exact in fp32, from the largest of them: the quotient 448 n / largest, with once more what it left
// out.  One on a border comes out as that, any other is 2^-21 or more away (448 n and border times largest have 24 bits at most).
struct RowCodesExact {
    float scale, by, part;  // part: largest / 448, exact
    DEV RowCodesExact(float largest, float rest)
    {
        constexpr float ONE_448TH = 1.0f / 448.0f;
        const float first = largest * ONE_448TH;
        bool normal;
        part = __builtin_fmaf(__builtin_fmaf(-first, 448.0f, largest), ONE_448TH, first);
        scale = row_scale(part * (8.0f / 7.0f) * rest, normal);
        by = normal ? 448.0f / largest : 0.0f;
    }
    template <int EPV, class F>
    DEV u32x2 codes(const float (&n)[EPV], F) const
    {
        u32 c[2] = {0, 0};
        float q[EPV];
#pragma unroll
        for (int i = 0; i < EPV; i++) {
            const float first = n[i] * by;
            q[i] = __builtin_fmaf(__builtin_fmaf(-first, part, n[i]), by, first);
        }
#pragma unroll
        for (int i = 0; i < EPV; i += 4) c[i / 4] = pack_fp8x4(q[i], q[i + 1], q[i + 2], q[i + 3]);
        return u32x2{c[0], c[1]};
    }
};
template <bool EXACT>
using RowCodesOf = std::conditional_t<EXACT, RowCodesExact, RowCodes>;

// EPV codes of a vector.
template <int EPV, bool NARROW>
DEV void store_codes(uint64_t row, const Piece &p, int cols, u32x2 c)
{
    if (!p.in) return;
    if (NARROW) store_bytes(row + (u32)p.at, (u32)cols, u32x4{c.x, c.y, 0, 0});
    else if constexpr (EPV == 8) *as_global<u32x2_a1>(row + (u32)p.at) = c;
    else *as_global<u32_a1>(row + (u32)p.at) = c.x;
}

// One team of TEAM lanes to a row, which stays in its registers: memory is read and written once, and bounds it.  8192x4096 bf16
// with a residual 44 us (268 MB, 6.1 TB/s), to 8 bits 40 (235 MB, 5.9); 163840x128 fp16 15.2 (84 MB, 5.5); one row 2.7 (3.1 a launch among ten).
template <class T, int TEAM, int NV, bool NARROW, bool WIDE, bool FP8>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void k_rms_norm(const NormArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = TEAM > 256 ? 1 : 256 / TEAM;
    // products of two 16-bit numbers are exact, those of bf16 448 times too; kept in registers where these leave eight wavefronts to a unit
    constexpr bool LOW = ESZ == 4 || WIDE, EXACT = !LOW && std::is_same<T, bf16_tag>::value, KEEP = NV * EPV <= 16;
    __shared__ float lds[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    const int lane = threadIdx.x % TEAM;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (row >= a.rows) return;  // a whole team; teams of several wavefronts are whole workgroups
    const uint64_t px = row_at(a.x, row, a.x_stride, a.x_group, a.x_group_stride, a.rows), pr = a.residual + (uint64_t)(row * a.residual_stride);
    const uint64_t at = (uint64_t)(row * a.cols) * ESZ;

    Piece piece[NV];
    u32x4 raw[NV], res[NV];
    Weights<T, NARROW, WIDE> weights[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        piece[v] = piece_of<EPV, NARROW>((v * TEAM + lane) * EPV, a.cols);
        raw[v] = load_row<ESZ, NARROW>(px, piece[v], a.cols);
    }
    if (a.residual) {
#pragma unroll
        for (int v = 0; v < NV; v++) res[v] = load_row<ESZ, NARROW>(pr, piece[v], a.cols);
    }
#pragma unroll
    for (int v = 0; v < NV; v++) weights[v].load(a.weight, piece[v], a.cols);
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        float f[EPV];
        Elem<T>::unpack(raw[v], f);
        if (a.residual) {
            float r[EPV];
            Elem<T>::unpack(res[v], r);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] += r[i];
            raw[v] = Elem<T>::pack(f);
            store_row<ESZ, NARROW>(a.h + at, piece[v], a.cols, raw[v]);
            Elem<T>::unpack(raw[v], f);
        }
        if (!NARROW) count_once(f, piece[v]);
#pragma unroll
        for (int i = 0; i < EPV; i++) sum = __builtin_fmaf(f[i], f[i], sum);
    }
    const float r = inverse_root(team_sum<TEAM>(sum, lds) * a.inv_cols, a.eps);
    if constexpr (FP8) {
        float unit, rest, mine = 0.0f;
        split_root(r, unit, rest);
        if (EXACT) unit *= 0.875f;
        float kept[KEEP ? NV : 1][EPV];
        auto again = [&] { if (!KEEP) asm("" : "+v"(unit)); };  // else they are made again, not kept by the compiler
        auto products = [&](int v, float (&p)[EPV]) {
            float f[EPV], w[EPV];
            Elem<T>::unpack(raw[v], f);
            weights[v].unpack(a.weight, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) p[i] = f[i] * unit * w[i];
        };
        // of one that is not 0, and so in the row; fp32 weights of two 16-bit vectors, 16 registers, are read again instead of kept (2048x16384
        // bf16 with a residual 46 us, 57 with 74 registers, 74 with spills)
        auto factors = [&](int v, int i, float &f, float &w) {
            float all[EPV];
            Elem<T>::unpack(raw[v], all);
            f = all[i] * unit;
            if (WIDE && NV == 2) w = as_global<const float>(a.weight)[piece[v].at + i];
            else {
                weights[v].unpack(a.weight, all);
                w = all[i];
            }
        };
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float(&p)[EPV] = kept[KEEP ? v : 0];
            products(v, p);
#pragma unroll
            for (int i = 0; i < EPV; i++) mine = fmaxf(mine, __builtin_fabsf(p[i]));
        }
        std::conditional_t<LOW, double, float> most;
        again();
        if constexpr (LOW) {
            most = team_largest_product<TEAM>(mine, lds, [&](float high) {
                float low = -__builtin_inff();
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    float(&p)[EPV] = kept[KEEP ? v : 0];
                    if (!KEEP) products(v, p);
#pragma unroll
                    for (int i = 0; i < EPV; i++)
                        if (__builtin_fabsf(p[i]) == high) {
                            float f, w;
                            factors(v, i, f, w);
                            low = fmaxf(low, __builtin_fmaf(__builtin_fabsf(f), __builtin_fabsf(w), -high));
                        }
                }
                return low;
            });
        } else most = team_largest<TEAM>(mine, lds);
        const RowCodesOf<EXACT> row_codes(most, rest);
        again();
        if (lane == 0) as_global<float>(a.scales)[row] = row_codes.scale;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float(&p)[EPV] = kept[KEEP ? v : 0];
            if (!KEEP) products(v, p);
            const u32x2 codes = row_codes.codes(p, [&](int at) {
                float f, w;
                factors(v, at, f, w);
                return (double)f * w;
            });
            store_codes<EPV, NARROW>(a.codes + (uint64_t)(row * a.cols), piece[v], a.cols, codes);
        }
        return;
    }
#pragma unroll
    for (int v = 0; v < NV; v++) {
        float f[EPV], w[EPV];
        Elem<T>::unpack(raw[v], f);
        weights[v].unpack(a.weight, w);
#pragma unroll
        for (int i = 0; i < EPV; i++) f[i] = f[i] * r * w[i];
        store_row<ESZ, NARROW>(a.y + at, piece[v], a.cols, Elem<T>::pack(f));
    }
}

// Rows too long for the registers of a workgroup: its 1024 lanes go over the row two or three times, behind the
// first time in h (or x), which the caches may still have.
template <class T, bool WIDE, bool FP8>
__global__ __launch_bounds__(1024) void k_rms_norm_long(const NormArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, STEP = 1024 * EPV;
    constexpr bool LOW = ESZ == 4 || WIDE, EXACT = !LOW && std::is_same<T, bf16_tag>::value;
    __shared__ float lds[32];
    const int64_t row = a.row0 + blockIdx.x;
    const uint64_t px = row_at(a.x, row, a.x_stride, a.x_group, a.x_group_stride, a.rows), pr = a.residual + (uint64_t)(row * a.residual_stride);
    const uint64_t at = (uint64_t)(row * a.cols) * ESZ, again = a.residual ? a.h + at : px;
    float sum = 0.0f;
    for (int col = threadIdx.x * EPV; col < a.cols; col += STEP) {
        const Piece p = piece_of<EPV, false>(col, a.cols);
        u32x4 raw = load_row<ESZ, false, false>(px, p, a.cols), res = {0, 0, 0, 0};
        if (a.residual) res = load_row<ESZ, false>(pr, p, a.cols);
        float f[EPV];
        Elem<T>::unpack(raw, f);
        if (a.residual) {
            float r[EPV];
            Elem<T>::unpack(res, r);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] += r[i];
            raw = Elem<T>::pack(f);
            store_row<ESZ, false, false>(a.h + at, p, a.cols, raw);
            Elem<T>::unpack(raw, f);
        }
        count_once(f, p);
#pragma unroll
        for (int i = 0; i < EPV; i++) sum = __builtin_fmaf(f[i], f[i], sum);
    }
    const float r = inverse_root(team_sum<1024>(sum, lds) * a.inv_cols, a.eps);
    // every lane reads back the vectors that it wrote itself: its own stores come before its own loads
    auto scaled = [&](const Piece &p, float by, float (&f)[EPV], float (&w)[EPV]) {
        const u32x4 raw = load_row<ESZ, false, false>(again, p, a.cols);
        Weights<T, false, WIDE> weights;
        weights.load(a.weight, p, a.cols);
        weights.unpack(a.weight, w);
        Elem<T>::unpack(raw, f);
#pragma unroll
        for (int i = 0; i < EPV; i++) f[i] *= by;
    };
    if constexpr (FP8) {
        float unit, rest, mine = 0.0f, f[EPV], w[EPV], p[EPV];
        split_root(r, unit, rest);
        if (EXACT) unit *= 0.875f;
        for (int col = threadIdx.x * EPV; col < a.cols; col += STEP) {
            scaled(piece_of<EPV, false>(col, a.cols), unit, f, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) mine = fmaxf(mine, __builtin_fabsf(f[i] * w[i]));
        }
        std::conditional_t<LOW, double, float> most;
        if constexpr (LOW) {
            most = team_largest_product<1024>(mine, lds, [&](float high) {
                float low = -__builtin_inff();
                for (int col = threadIdx.x * EPV; col < a.cols; col += STEP) {
                    scaled(piece_of<EPV, false>(col, a.cols), unit, f, w);
#pragma unroll
                    for (int i = 0; i < EPV; i++)
                        if (__builtin_fabsf(f[i] * w[i]) == high) low = fmaxf(low, __builtin_fmaf(__builtin_fabsf(f[i]), __builtin_fabsf(w[i]), -high));
                }
                return low;
            });
        } else most = team_largest<1024>(mine, lds);
        const RowCodesOf<EXACT> row_codes(most, rest);
        if (threadIdx.x == 0) as_global<float>(a.scales)[row] = row_codes.scale;
        for (int col = threadIdx.x * EPV; col < a.cols; col += STEP) {
            const Piece here = piece_of<EPV, false>(col, a.cols);
            scaled(here, unit, f, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) p[i] = f[i] * w[i];
            store_codes<EPV, false>(a.codes + (uint64_t)(row * a.cols), here, a.cols, row_codes.codes(p, [&](int at) { return (double)f[at] * w[at]; }));
        }
    } else {
        for (int col = threadIdx.x * EPV; col < a.cols; col += STEP) {
            const Piece p = piece_of<EPV, false>(col, a.cols);
            float f[EPV], w[EPV];
            scaled(p, r, f, w);
#pragma unroll
            for (int i = 0; i < EPV; i++) f[i] *= w[i];
            store_row<ESZ, false>(a.y + at, p, a.cols, Elem<T>::pack(f));
        }
    }
}

struct NormBackwardArgs {
    uint64_t dy, dh, h, weight, dx, sums;  // dh, weight, dx, sums: 0 for none.  sums: fp32 [workgroups][sums_stride(cols)]
    int64_t h_stride, h_group_stride;      // bytes; all others are contiguous
    u32 h_group;
    int64_t rows;
    int cols;
    float eps, inv_cols;
};

// A team goes over every (teams in the grid)-th row, one after the other, and keeps its part of dw in registers;
// a workgroup's teams add theirs up in LDS and leave a row of fp32 sums, which k_column_sums adds up.  8192x4096 bf16 with the
// residual's gradient 46.5 us (268 MB, 5.8 TB/s) and 3.9 for the sums, 163840x128 fp16 23.6 (126 MB, 5.3) and 3.8.
template <class T, int TEAM, int NV, bool NARROW, bool WIDE>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void k_rms_norm_backward(const NormBackwardArgs a)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = TEAM > 256 ? 1 : 256 / TEAM;
    __shared__ float lds[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    __shared__ float add[TEAMS > 1 ? 256 * NV * EPV : 1];
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    float acc[NV][EPV];
    Piece piece[NV];
    Weights<T, NARROW, WIDE> weights[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        piece[v] = piece_of<EPV, NARROW>((v * TEAM + lane) * EPV, a.cols);
        weights[v].load(a.weight, piece[v], a.cols);
#pragma unroll
        for (int i = 0; i < EPV; i++) acc[v][i] = 0.0f;
    }

    // the next row is on its way while this one is worked on, where there are registers for it
    constexpr bool AHEAD = TEAM * NV * EPV <= 8192;
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    u32x4 dy_next[NV], h_next[NV], dh_next[NV];
    auto fetch = [&](int64_t row) {
        if (AHEAD && row >= a.rows) return;
        const uint64_t at = (uint64_t)(row * a.cols) * ESZ, ph = row_at(a.h, row, a.h_stride, a.h_group, a.h_group_stride, a.rows);
#pragma unroll
        for (int v = 0; v < NV; v++) dy_next[v] = load_row<ESZ, NARROW>(a.dy + at, piece[v], a.cols);
#pragma unroll
        for (int v = 0; v < NV; v++) h_next[v] = load_row<ESZ, NARROW>(ph, piece[v], a.cols);
        if (a.dh) {
#pragma unroll
            for (int v = 0; v < NV; v++) dh_next[v] = load_row<ESZ, NARROW>(a.dh + at, piece[v], a.cols);
        }
    };
    int64_t row = (int64_t)blockIdx.x * TEAMS + team;
    if (AHEAD) fetch(row);
    for (; row < a.rows; row += step) {
        if (!AHEAD) fetch(row);
        const uint64_t at = (uint64_t)(row * a.cols) * ESZ;
        u32x4 dy[NV], h[NV], dh[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            dy[v] = dy_next[v];
            h[v] = h_next[v];
            dh[v] = dh_next[v];
        }
        if (AHEAD) fetch(row + step);
        float squares = 0.0f, along = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            float f[EPV], g[EPV], w[EPV];
            Elem<T>::unpack(h[v], f);
            Elem<T>::unpack(dy[v], g);
            weights[v].unpack(a.weight, w);
            if (!NARROW) {
                count_once(f, piece[v]);
                count_once(g, piece[v]);
            }
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
            weights[v].unpack(a.weight, w);
            if (a.dh) Elem<T>::unpack(dh[v], d);
#pragma unroll
            for (int i = 0; i < EPV; i++) {
                acc[v][i] = __builtin_fmaf(g[i], f[i] * r, acc[v][i]);
                f[i] = r * (g[i] * w[i] - f[i] * c);
                if (a.dh) f[i] += d[i];
            }
            if (a.dx) store_row<ESZ, NARROW>(a.dx + at, piece[v], a.cols, Elem<T>::pack(f));
        }
    }
    if (!a.sums) return;
    const uint64_t sums = a.sums + (uint64_t)blockIdx.x * (uint64_t)sums_stride(a.cols) * 4;
    if constexpr (TEAMS > 1) {
        constexpr int WIDTH = NV * TEAM * EPV;  // [team][vector][element][lane]
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int i = 0; i < EPV; i++) add[team * WIDTH + (v * EPV + i) * TEAM + lane] = acc[v][i];
        __syncthreads();
        for (int c = threadIdx.x; c < WIDTH; c += 256) {
            float s = 0.0f;
#pragma unroll 4
            for (int t = 0; t < TEAMS; t++) s += add[t * WIDTH + c];
            const int v = c / (EPV * TEAM), e = c / TEAM % EPV, l = c % TEAM;
            const Piece p = piece_of<EPV, NARROW>((v * TEAM + l) * EPV, a.cols);
            if (p.in) as_global<float>(sums)[p.at + e] = s;
        }
    } else {
#pragma unroll
        for (int v = 0; v < NV; v++) store_sums(sums, piece[v], acc[v]);
    }
}

// Rows too long for that: first r and c of every row, then dx and the sums, a workgroup to 256 vectors of columns
// and a share of the rows, four rows at a time.
template <class T, bool WIDE>
__global__ __launch_bounds__(1024) void k_rms_norm_backward_long(const NormBackwardArgs a, uint64_t factors)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, U = 2, STEP = 1024 * EPV;
    __shared__ float lds[32];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t at = (uint64_t)(row * a.cols) * ESZ, ph = row_at(a.h, row, a.h_stride, a.h_group, a.h_group_stride, a.rows);
        float squares = 0.0f, along = 0.0f;
        for (int col = threadIdx.x * EPV; col < a.cols; col += U * STEP) {
            Weights<T, false, WIDE> weights[U];
            Piece p[U];
            u32x4 h[U], dy[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                p[u] = piece_of<EPV, false>(col + u * STEP, a.cols);
                h[u] = load_row<ESZ, false, false>(ph, p[u], a.cols);
                dy[u] = load_row<ESZ, false, false>(a.dy + at, p[u], a.cols);
                weights[u].load(a.weight, p[u], a.cols);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                float f[EPV], g[EPV], w[EPV];
                weights[u].unpack(a.weight, w);
                Elem<T>::unpack(h[u], f);
                Elem<T>::unpack(dy[u], g);
                count_once(f, p[u]);
                count_once(g, p[u]);
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
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void k_rms_norm_backward_columns(const NormBackwardArgs a, uint64_t factors)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, U = 4;
    const Piece p = piece_of<EPV, false>((int)(blockIdx.x * 256 + threadIdx.x) * EPV, a.cols);
    if (!p.in) return;
    float acc[EPV] = {}, w[EPV];
    Weights<T, false, WIDE> weights;
    weights.load(a.weight, p, a.cols);
    weights.unpack(a.weight, w);
    for (int64_t first = (int64_t)blockIdx.y * U; first < a.rows; first += (int64_t)gridDim.y * U) {
        u32x4 h[U], dy[U], dh[U];
        float r[U], c[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t row = first + u < a.rows ? first + u : a.rows - 1;
            const uint64_t at = (uint64_t)(row * a.cols) * ESZ;
            h[u] = load_row<ESZ, false>(row_at(a.h, row, a.h_stride, a.h_group, a.h_group_stride, a.rows), p, a.cols);
            dy[u] = load_row<ESZ, false>(a.dy + at, p, a.cols);
            if (a.dh) dh[u] = load_row<ESZ, false>(a.dh + at, p, a.cols);
            r[u] = as_global<const float>(factors)[2 * row];
            c[u] = as_global<const float>(factors)[2 * row + 1];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (first + u >= a.rows) continue;
            float f[EPV], g[EPV], d[EPV];
            Elem<T>::unpack(h[u], f);
            Elem<T>::unpack(dy[u], g);
            if (a.dh) Elem<T>::unpack(dh[u], d);
#pragma unroll
            for (int i = 0; i < EPV; i++) {
                acc[i] = __builtin_fmaf(g[i], f[i] * r[u], acc[i]);
                f[i] = r[u] * (g[i] * w[i] - f[i] * c[u]);
                if (a.dh) f[i] += d[i];
            }
            if (a.dx) store_row<ESZ, false>(a.dx + (uint64_t)((first + u) * a.cols) * ESZ, p, a.cols, Elem<T>::pack(f));
        }
    }
    if (a.sums) store_sums(a.sums + (uint64_t)blockIdx.y * (uint64_t)sums_stride(a.cols) * 4, p, acc);
}

// out[c] = the sum of sums[p][c] over p, rounded once: 4 lanes to 16 columns, 64 of the parts side by side.
template <class T>
__global__ __launch_bounds__(256) void k_column_sums(uint64_t sums, int64_t parts, int cols, uint64_t out)
{
    __shared__ float add[64][17];
    const int64_t stride = sums_stride(cols);
    const int lane = threadIdx.x & 3, group = threadIdx.x >> 2;
    const int64_t col = (int64_t)blockIdx.x * 16 + lane * 4;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col < stride) {
#pragma unroll 8
        for (int64_t p = group; p < parts; p += 64) {
            const u32x4 v = *as_global<const u32x4>(sums + (uint64_t)(p * stride + col) * 4);
#pragma unroll
            for (int i = 0; i < 4; i++) s[i] += as_f(v[i]);
        }
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

// The values of 8-bit rows, a lane for EPV of them.  8192x4096 to bf16 15.1 us (101 MB, 6.7 TB/s).
template <class T, int TEAM, bool NARROW>
__global__ __launch_bounds__(256) void k_fp8_rows(uint64_t codes, uint64_t scales, int64_t row0, int64_t rows, int cols, uint64_t out)
{
    constexpr int ESZ = Elem<T>::ESZ, EPV = Elem<T>::EPV, TEAMS = 256 / TEAM, U = 2;
    const int64_t row = row0 + (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (row >= rows) return;
    const float scale = as_global<const float>(scales)[row];
    const uint64_t from = codes + (uint64_t)(row * cols), to = out + (uint64_t)(row * cols) * ESZ;
    for (int col = threadIdx.x % TEAM * EPV; col < cols; col += U * TEAM * EPV) {
        u32 w[U][2] = {};
        Piece p[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            p[u] = piece_of<EPV, NARROW>(col + u * TEAM * EPV, cols);
            if (!p[u].in) continue;
            const uint64_t at = from + (u32)p[u].at;
            if (NARROW) {
                const u32x4 v = load_bytes(at, (u32)cols);
                w[u][0] = v.x;
                w[u][1] = v.y;
            } else if constexpr (EPV == 8) {
                const u32x2 v = LOAD_STREAM(as_global<const u32x2_a1>(at));
                w[u][0] = v.x;
                w[u][1] = v.y;
            } else w[u][0] = LOAD_STREAM(as_global<const u32_a1>(at));
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
            store_row<ESZ, NARROW>(to, p[u], cols, Elem<T>::pack(f));
        }
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Lanes and vectors to a row of `vectors`; {0, 0}: too long for registers.  Two vectors a lane hide more of memory's latency
// than one, and lanes that a row leaves idle cost as much as others: rows of 16 vectors (163840 fp16) took 17.5 us with 8 lanes of
// two, 18.4 with 16, 47 with 64; rows of 512 (8192 bf16 with a residual) 45.8 with 512 lanes, 47.5 with 256 of two, one
// row 3.4 and 3.8.  Now 15.5, 44.1 (6.1 TB/s) and 3.1.
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
// one, 52.9 with 256 of two; of 2048 (2048 bf16) 71 with 1024 of two, 121 with 512 of four, which spill.  Now 43, 28, 49, 50
// and 71: 4.0, 4.7, 5.5, 5.3 and 3.8 TB/s.
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
    if (vectors <= 2048) return {1024, 2};
    return {0, 0};
}

static bool narrow_row(int64_t cols, int size) { return cols * size < 16; }

#define SHAPE(TEAM, NV) case TEAM * 16 + NV: K(TEAM, NV, false); break;

template <class T, bool WIDE, bool FP8>
static int norm(NormArgs a, hipStream_t st)
{
    RowShape shape = norm_shape((a.cols + Elem<T>::EPV - 1) / Elem<T>::EPV);
    if (WIDE && FP8 && shape.nv == 4) shape = {0, 0};  // too long with fp32 weights: 1024x32768 bf16 34 us, with a residual 58, 67 with spills; 1600x20000 55, 57
    const void *k = (const void *)k_rms_norm_long<T, WIDE, FP8>;
#define K(TEAM, NV, NARROW) k = (const void *)k_rms_norm<T, TEAM, NV, NARROW, WIDE, FP8>
    switch (shape.team * 16 + shape.nv) {
        SHAPE(8, 1) SHAPE(8, 2) SHAPE(16, 2) SHAPE(32, 2) SHAPE(64, 2) SHAPE(256, 1) SHAPE(512, 1) SHAPE(512, 2) SHAPE(1024, 2)
    }
    if constexpr (!(WIDE && FP8))
        if (shape.nv == 4) K(1024, 4, false);
    if (narrow_row(a.cols, Elem<T>::ESZ)) K(8, 1, true);
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

template <class T, bool WIDE>
static int norm_backward(NormBackwardArgs a, uint64_t factors, int64_t parts, hipStream_t st)
{
    const RowShape shape = norm_backward_shape((a.cols + Elem<T>::EPV - 1) / Elem<T>::EPV, Elem<T>::ESZ);
    if (shape.team == 0) {
        void *args[] = {(void *)&a, (void *)&factors};
        int rc = (int)hipLaunchKernel((const void *)k_rms_norm_backward_long<T, WIDE>, dim3((unsigned)std::min<int64_t>(a.rows, 2048)), dim3(1024),
                                      args, 0, st);
        if (rc) return rc;
        const unsigned across = (unsigned)((a.cols + 256 * Elem<T>::EPV - 1) / (256 * Elem<T>::EPV));
        return (int)hipLaunchKernel((const void *)k_rms_norm_backward_columns<T, WIDE>, dim3(across, (unsigned)parts), dim3(256), args, 0, st);
    }
    const void *k = nullptr;
#define K(TEAM, NV, NARROW) k = (const void *)k_rms_norm_backward<T, TEAM, NV, NARROW, WIDE>
    if constexpr (Elem<T>::ESZ == 4) {
        if (shape.team == 64 && shape.nv == 4) K(64, 4, false);
    } else if (shape.team == 256) K(256, 1, false);
    switch (shape.team * 16 + shape.nv) {
        SHAPE(8, 1) SHAPE(8, 2) SHAPE(16, 2) SHAPE(16, 3) SHAPE(32, 2) SHAPE(64, 2) SHAPE(64, 3) SHAPE(512, 1) SHAPE(512, 2) SHAPE(1024, 2)
    }
    if (narrow_row(a.cols, Elem<T>::ESZ)) K(8, 1, true);
#undef K
#undef SHAPE
    void *args[] = {(void *)&a};
    return (int)hipLaunchKernel(k, dim3((unsigned)parts), dim3(shape.team > 256 ? shape.team : 256), args, 0, st);
}

static bool groups_ok(int64_t rows, int64_t cols, int64_t stride, int64_t group, int64_t group_stride)
{
    return group >= 1 && group <= ROWS_MOST && stride >= (group > 1 && rows > 1 ? cols : 0) && group_stride >= (rows > group ? cols : 0);
}

extern "C" int tftq_rms_norm(int dtype, int weight_dtype, const void *x, int64_t x_stride, int64_t x_group, int64_t x_group_stride,
                             const void *residual, int64_t residual_stride, const void *weight, int64_t rows, int64_t cols, float eps, void *h, void *y, void *codes, float *scales,
                             int device, void *stream)
{
    if (!dtype_ok(dtype) || (weight && weight_dtype != dtype && weight_dtype != TFTQ_F32)) return TFTQ_E_DTYPE;
    if (!rows_ok(rows, cols)) return TFTQ_E_SHAPE;
    if (rows == 0 || cols == 0) return 0;
    if (!x || !residual != !h || !codes != !scales || !y == !codes || !(eps >= 0.0f)) return TFTQ_E_ARG;
    if (!groups_ok(rows, cols, x_stride, x_group, x_group_stride) || (residual && residual_stride < (rows > 1 ? cols : 0))) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    const int size = dtype_size(dtype);
    const NormArgs a = {(uint64_t)x, (uint64_t)residual, (uint64_t)weight, (uint64_t)y, (uint64_t)h, (uint64_t)codes, (uint64_t)scales,
                        x_stride * size, residual_stride * size, x_group_stride * size, (u32)x_group, 0, rows, (int)cols, eps, 1.0f / (float)cols};
    hipStream_t st = (hipStream_t)stream;
    const bool wide = weight && weight_dtype != dtype;
#define NORM(T) (wide ? codes ? norm<T, true, true>(a, st) : norm<T, true, false>(a, st) : codes ? norm<T, false, true>(a, st) : norm<T, false, false>(a, st))
    if (dtype == TFTQ_F32) return codes ? norm<float, false, true>(a, st) : norm<float, false, false>(a, st);
    return dtype == TFTQ_F16 ? NORM(f16_tag) : NORM(bf16_tag);
#undef NORM
}

extern "C" int64_t tftq_rms_norm_backward_workspace(int dtype, int64_t rows, int64_t cols)
{
    if (!dtype_ok(dtype)) return TFTQ_E_DTYPE;
    if (!rows_ok(rows, cols)) return TFTQ_E_SHAPE;
    if (rows == 0 || cols == 0) return 0;
    return norm_parts(rows, cols, dtype_size(dtype)) * sums_stride(cols) * 4 + rows * 8;
}

extern "C" int tftq_rms_norm_backward(int dtype, int weight_dtype, const void *dy, const void *dh, const void *h, int64_t h_stride,
                                      int64_t h_group, int64_t h_group_stride, const void *weight, int64_t rows, int64_t cols, float eps, void *dx, void *dweight, void *workspace,
                                      int64_t workspace_bytes, int device, void *stream)
{
    if (!dtype_ok(dtype) || (weight && weight_dtype != dtype && weight_dtype != TFTQ_F32)) return TFTQ_E_DTYPE;
    if (!rows_ok(rows, cols)) return TFTQ_E_SHAPE;
    if (cols == 0 || (rows == 0 && !dweight)) return 0;
    if ((dweight && !weight) || (rows && (!dy || !h || !workspace || ((uintptr_t)workspace & 15))) || (!dx && !dweight) || !(eps >= 0.0f)) return TFTQ_E_ARG;
    if (rows && !groups_ok(rows, cols, h_stride, h_group, h_group_stride)) return TFTQ_E_ARG;
    const int size = dtype_size(dtype);
    const int64_t parts = rows ? norm_parts(rows, cols, size) : 0, sums = parts * sums_stride(cols) * 4;
    if (rows && workspace_bytes < sums + rows * 8) return TFTQ_E_SIZE;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    hipStream_t st = (hipStream_t)stream;
    if (rows) {
        const NormBackwardArgs a = {(uint64_t)dy, (uint64_t)dh, (uint64_t)h, (uint64_t)weight, (uint64_t)dx, dweight ? (uint64_t)workspace : 0,
                                    h_stride * size, h_group_stride * size, (u32)h_group, rows, (int)cols, eps, 1.0f / (float)cols};
        const uint64_t factors = (uint64_t)workspace + (uint64_t)sums;
        const bool wide = weight && weight_dtype != dtype;
#define NORM(T) (wide ? norm_backward<T, true>(a, factors, parts, st) : norm_backward<T, false>(a, factors, parts, st))
        const int rc = dtype == TFTQ_F32 ? norm_backward<float, false>(a, factors, parts, st) : dtype == TFTQ_F16 ? NORM(f16_tag) : NORM(bf16_tag);
#undef NORM
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
#define K(T)                                                                                  \
    (narrow_row(cols, Elem<T>::ESZ) ? (const void *)k_fp8_rows<T, 8, true>                        \
     : team == 8                    ? (const void *)k_fp8_rows<T, 8, false>                       \
     : team == 64                   ? (const void *)k_fp8_rows<T, 64, false>                      \
                                    : (const void *)k_fp8_rows<T, 256, false>)
    const void *k = dtype == TFTQ_F32 ? K(float) : dtype == TFTQ_F16 ? K(f16_tag) : K(bf16_tag);
#undef K
    const int64_t at_once = ROWS_THREADS / team;
    for (; row0 < rows; row0 += at_once)
        if (const int rc = (int)hipLaunchKernel(k, dim3((unsigned)((std::min(at_once, rows - row0) + teams - 1) / teams)), dim3(256), args, 0, (hipStream_t)stream))
            return rc;
    return 0;
}
