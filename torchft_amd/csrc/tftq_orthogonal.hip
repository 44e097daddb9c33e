// Newton-Schulz orthogonalisation of a list of matrices, with Muon's momentum before it and its update
// of the weights behind it, and the C entry of both.
//
//   X = u / max(|u|, eps);  T times:  A = X X^T,  X <- a X + (b A + c A A) X
//
// X has no more rows than columns (of a taller matrix the transpose is taken: the result is its
// transpose).  Per iteration three products on the 16-bit matrix cores, A, A A and B X, one launch
// each for all matrices of the list (up to NS_MOST at a time).
//
// What is rounded to 16 bits.  X, A and B are handed to the matrix cores as fp16 numbers, scaled by
// powers of two; sums are fp32.  Rounding A and B to 11 bits as they are loses most on their
// diagonals: A's eigenvalues tend to ~0.9, so its diagonal is by far its largest part, and an error of
// 2^-12 there is one of 2^-12 in all that follows.  So the diagonals are kept apart in fp32:
// A = D + E, B = F + G with E and G zero on the diagonal, and
//     (A A)[i][j] = (E E)[i][j] + (D[i] + D[j]) E[i][j],     (B X)[i][j] = F[i] X[i][j] + (G X)[i][j];
// and X keeps what its rounding leaves as a second fp16 number (22 bits together), which the products
// leave out and the term (a + F) X takes in.  (Not in the last iteration, to which it adds nothing that
// one rounding of the result would leave: errors 0 to 10 % larger, and 4 of 46 bytes an element less.)
// Relative error of the result against 64 bits, one product each, matrices of 64x64 to 1024x1024 with even, low-rank and 1/i spectra: 2.4e-4 to 1.3e-3
// (bf16 results are rounded by 1.7e-3; A, B and X in plain bf16: 1.3e-2 to 7.7e-2, in plain fp16 up to
// 9e-3; matrices of nearly rank one: ns_precise).  `precise`: A, B and X^T have second numbers too and every product is
// three, high x high + low x high + high x low: 5e-7 to 5e-6, where fp32 products give 1e-6 to 6e-6 (nearly rank one 5e-5
// to 3.4e-4, where they give 7e-5 to 3.8e-4), at three times the work
// of the 16-bit cores, which is a fifth of what the fp32 ones would take.
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and stored twice.
// X^T is stored beside X so that all three products contract rows of both operands (tftq_tile.h).
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

#include "tftq_device.h"
#include "tftq_tile.h"

typedef _Float16 ns_h8 __attribute__((ext_vector_type(8)));

constexpr int NS_MOST = 24;            // matrices of a launch: their descriptors travel in its arguments
constexpr int64_t NS_LONGEST = 1 << 24;  // rows or columns
// What X, E and G are scaled by at most: |X| <= ~1.2, |A| <= ~1.5, |B| <= ~3 with the usual coefficients, and fp16
// ends at 65504.  Of others the bounds of every iteration say how much less (NsScales).
// X of a gradient so small that eps divides it stays small: its scale is larger by a power of two (ns_scale).
constexpr float SCALE_X = 16384.f, SCALE_E = 4096.f, SCALE_G = 2048.f;
constexpr int NORM_COLS = 1024;
// The rows of the matrix as it lies, `wide` columns of at most 1024 each, whose squares a workgroup sums up:
// 64, or 8 where that makes no more than 1024 sums of a matrix (1001x130: 57 -> 12 us).
__host__ __device__ static inline int ns_part_rows(int64_t high, int64_t wide)
{
    return (high + 7) / 8 * ((wide + NORM_COLS - 1) / NORM_COLS) <= 1024 ? 8 : 64;
}
__host__ __device__ static inline int64_t ns_parts_of(int64_t high, int64_t wide)
{
    const int rows = ns_part_rows(high, wide);
    return (high + rows - 1) / rows * ((wide + NORM_COLS - 1) / NORM_COLS);
}

struct NsMatrix {
    const uint8_t *in;
    float *momentum;
    uint8_t *out;
    int64_t ld_in, ld_momentum, ld_out;
    uint8_t *work;
    int rows, cols;  // of X
    int flip;        // X is the transpose of the matrix as it lies
    float step;      // out = keep * out - step * X with NsParams::update, else out = X
    int pieces;      // the launch's workgroups of this matrix
    int splits;      // of them share a tile, each a part of its panels (NsSplit)
};
struct NsLaunch {
    int count;
    int first[NS_MOST];  // of every matrix the first workgroup (products: in eighths, ns_tile); past the last one INT_MAX
    NsMatrix m[NS_MOST];
};
struct NsParams {
    float momentum, keep, a, b, c, eps, growth;
    int nesterov, out_dtype, update;
    int last, next_last;  // the last iteration, the one before it
    // of this iteration (NsScales): X's scale in that of the first one, the next one's in this one's; E's; and
    // what the sums of A A, E and the sums of G X are multiplied by for G and X
    float x, x_next, e, per_ee, aa_to_g, c_to_g, b_to_g, gx_to_x;
};
static_assert(sizeof(NsLaunch) + sizeof(NsParams) <= 3800, "kernel arguments");

// The parts of a matrix's workspace.
struct NsWork {
    uint8_t *x, *xl;        // X and its remainder, panels of columns
    uint8_t *t, *t2, *tl, *tl2;  // X^T, of this iteration and of the next one (then the other way round)
    uint8_t *e, *el;        // A without its diagonal
    uint8_t *g, *gl;        // B without its diagonal
    float *d, *f;           // the diagonals
    float *scale;           // of X: SCALE_X, or more
    double *squares;        // of the parts of u
    int *tickets;           // of every tile that workgroups share: how many of them are done
    float *sums;            // theirs
    int64_t bytes;          // without `sums`
};
constexpr int NS_SHARED = 512;  // workgroups of a launch with shared tiles, at most (2 to a compute unit)
__host__ __device__ static __forceinline__ NsWork ns_work(uint8_t *base, int64_t r, int64_t k, int flip, bool precise)
{
    const int64_t rp = (r + 63) / 64, kp = (k + 63) / 64, x = kp * r * PANEL_BYTES, t = rp * k * PANEL_BYTES, a = rp * r * PANEL_BYTES;
    const int64_t high = flip ? k : r, wide = flip ? r : k;
    const int64_t parts = ns_parts_of(high, wide);
    NsWork w;
    w.x = base, w.xl = w.x + x;
    w.t = w.xl + x, w.t2 = w.t + t;
    w.tl = w.t2 + t, w.tl2 = w.tl + (precise ? t : 0);
    w.e = w.tl2 + (precise ? t : 0), w.g = w.e + a;
    w.el = w.g + a, w.gl = w.el + (precise ? a : 0);
    w.d = (float *)(w.gl + (precise ? a : 0)), w.f = w.d + ((r + 63) & ~63ll);
    w.scale = w.f + ((r + 63) & ~63ll);
    w.squares = (double *)(w.scale + 32);
    w.tickets = (int *)(w.squares + ((parts + 15) & ~15ll));
    w.sums = (float *)(w.tickets + NS_SHARED / 2);
    w.bytes = (uint8_t *)w.sums - base;
    return w;
}

// The matrix of this workgroup, and which of the matrix's workgroups it is.  A kernel's arguments may lie in
// host memory: all of `first` comes in one load (a search of 24 matrices that loads one at a time takes 8.0 us
// in an empty kernel, this one 2.8; 24 matrices of 128x256 orthogonalised: 218, 153), and `count`, the
// first argument, comes in registers.
__device__ static inline int ns_find(const NsLaunch &l, int count, int id, int *piece)
{
    int i = 0, start = 0;
    *piece = id;
    if (count == 1) return 0;
#pragma unroll
    for (int n = 1; n < NS_MOST; n++)
        if (id >= l.first[n]) i = n, start = l.first[n];
    *piece = id - start;
    return i;
}

// 4 neighbouring elements at any element's address, n of which exist.
typedef float ns_f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 ns_h4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 ns_b4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ static inline tile_f4 ns_read(const uint8_t *from, int64_t at, int dtype, int n)
{
    tile_f4 v = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        if (dtype == TFTQ_F32) return *(const ns_f4_any *)(from + at * 4);
        if (dtype == TFTQ_F16) return __builtin_convertvector(*(const ns_h4_any *)(from + at * 2), tile_f4);
        return __builtin_convertvector(*(const ns_b4_any *)(from + at * 2), tile_f4);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) v[i] = dtype == TFTQ_F32 ? ((const float *)from)[at + i] : dtype == TFTQ_F16 ? (float)((const _Float16 *)from)[at + i] : (float)((const __bf16 *)from)[at + i];
    return v;
}
// The same of one type, 4 elements that all exist: loads of several of them, without a branch between, go out together.
template <int DTYPE>
__device__ static inline tile_f4 ns_read4(const uint8_t *from, int64_t at)
{
    if constexpr (DTYPE == TFTQ_F32) return *(const ns_f4_any *)(from + at * 4);
    else if constexpr (DTYPE == TFTQ_F16) return __builtin_convertvector(*(const ns_h4_any *)(from + at * 2), tile_f4);
    else return __builtin_convertvector(*(const ns_b4_any *)(from + at * 2), tile_f4);
}
// The matrix and the tile of a product's workgroup: every XCD takes an eighth of every matrix's tiles,
// neighbouring ones (workgroups go to the 8 XCDs in turn), so that the matrices with most panels are
// shared by all (one run of the whole list's tiles each: A of 3 matrices of 88 panels and 4 of 32, 161 us).
// False for a workgroup that fills up a matrix's last eight.
__device__ static __forceinline__ bool ns_tile(const NsLaunch &l, int matrices, int id, int *matrix, int *piece)
{
    int n;
    *matrix = ns_find(l, matrices, id >> 3, &n);
    const int xcd = id & 7, count = l.m[*matrix].pieces, whole = count >> 3, more = count & 7;
    *piece = xcd * whole + min(xcd, more) + n;
    return n < whole + (xcd < more);
}

// The momentum's next value and the update that is orthogonalised, g + momentum (m - g) as a sum of two
// products: where m is mostly the same gradient the difference would cancel to a tenth of g, and what its
// rounding leaves in directions that are weak in u comes out up to a^5 (480) times as large.
__device__ static inline float ns_momentum(float m, float g, const NsParams &p) { return m * p.momentum + (1.f - p.momentum) * g; }
__device__ static inline float ns_update(float m, float g, const NsParams &p) { return p.nesterov ? m * p.momentum + (1.f - p.momentum) * g : m; }

// momentum <- its next value; the sums of the squares of u, one for 8 or 64 rows of 1024, in 64 bits: no
// gradient's norm leaves their range, and the order of the additions is always the same.  Bound by memory:
// 4096x14336 bf16 36 us (117 MB, 3.2 TB/s), 44 M elements with momentum 84 us (440 MB, 5.2 TB/s).  A branch on
// the type or the row's end at every load makes each wait for the one before (55 and 154 us).
template <int DTYPE, bool MOMENTUM>
__global__ __launch_bounds__(256) void k_ns_squares(int count, int precise, const NsLaunch l, const NsParams p)
{
    __shared__ double sums[4];
    int piece;
    const NsMatrix m = l.m[ns_find(l, count, blockIdx.x, &piece)];
    const int high = m.flip ? m.cols : m.rows, wide = m.flip ? m.rows : m.cols;
    const int across = (wide + NORM_COLS - 1) / NORM_COLS;
    const int part = ns_part_rows(high, wide);
    const int row0 = piece / across * part, col0 = piece % across * NORM_COLS;
    const int rows = min(part, high - row0);
    // a thread has 4 neighbouring columns of every `apart`th row
    const int groups = (min(NORM_COLS, wide - col0) + 3) >> 2, apart = 256 / groups;
    const int c = col0 + (int)threadIdx.x % groups * 4, n = wide - c;
    double sum = 0;
    constexpr int AT_ONCE = 8;  // rows whose loads are in flight together
    auto add = [&](auto whole) {
        for (int r0 = row0 + (int)threadIdx.x / groups; r0 < row0 + rows; r0 += AT_ONCE * apart) {
            tile_f4 u[AT_ONCE], next[AT_ONCE];
#pragma unroll
            for (int q = 0; q < AT_ONCE; q++) {
                const int64_t r = min(r0 + q * apart, row0 + rows - 1);
                u[q] = whole ? ns_read4<DTYPE>(m.in, r * m.ld_in + c) : ns_read(m.in, r * m.ld_in + c, DTYPE, n);
                if (MOMENTUM)
                    next[q] = whole ? ns_read4<TFTQ_F32>((const uint8_t *)m.momentum, r * m.ld_momentum + c)
                                    : ns_read((const uint8_t *)m.momentum, r * m.ld_momentum + c, TFTQ_F32, n);
            }
#pragma unroll
            for (int q = 0; q < AT_ONCE; q++) {
                const int64_t r = r0 + q * apart;
                if (r >= row0 + rows) continue;
                if (MOMENTUM) {
                    float *at = m.momentum + r * m.ld_momentum + c;
#pragma unroll
                    for (int i = 0; i < 4; i++) next[q][i] = ns_momentum(next[q][i], u[q][i], p), u[q][i] = ns_update(next[q][i], u[q][i], p);
                    if (whole) {
                        *(ns_f4_any *)at = next[q];
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (i < n) at[i] = next[q][i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) sum += (double)u[q][i] * (double)u[q][i];
            }
        }
    };
    if ((int)threadIdx.x < groups * apart) {
        if (n >= 4) add(std::true_type());
        else add(std::false_type());
    }
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) ns_work(m.work, m.rows, m.cols, m.flip, precise).squares[piece] = sums[0] + sums[1] + sums[2] + sums[3];
}

// What X is scaled by.  |X| starts as norm / eps if that is less than 1 and grows by |a| per iteration at
// most while it is small (`growth` in all): the power of two that this leaves room for.
__device__ static inline float ns_scale(double norm, const NsParams &p)
{
    const double room = (double)p.eps / (norm * p.growth);
    return room > 1.0 && room < 1e30 ? ldexpf(SCALE_X, ilogb(room)) : SCALE_X;
}

// v * scale as two fp16 numbers.
__device__ static inline void ns_split(float v, float scale, _Float16 *high, _Float16 *low)
{
    *high = (_Float16)(v * scale);
    *low = (_Float16)(v * scale - (float)*high);
}

// X and X^T in panels from u / |u|, a square of 64 per workgroup, turned in LDS.  Bound by memory: 4096x14336 bf16
// 100 us (470 MB, 4.7 TB/s).
template <int DTYPE, bool MOMENTUM>
__global__ __launch_bounds__(256) void k_ns_start(int count, int precise, const NsLaunch l, const NsParams p)
{
    __shared__ float tile[64][65];
    __shared__ double sums[4];
    int piece;
    const NsMatrix m = l.m[ns_find(l, count, blockIdx.x, &piece)];
    const NsWork w = ns_work(m.work, m.rows, m.cols, m.flip, precise);
    const int across = (m.cols + 63) / 64;
    const int row0 = piece / across * 64, col0 = piece % across * 64;
    const int high = m.flip ? m.cols : m.rows, wide = m.flip ? m.rows : m.cols;
    // read along the rows of the matrix as it lies, on the way while the norm is added up
    const int at_row = m.flip ? col0 : row0, at_col = m.flip ? row0 : col0;
    const bool inside = at_row + 64 <= high && at_col + 64 <= wide;
    tile_f4 v[4] = {}, old[4] = {};
    if (inside) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t row = at_row + ((int)threadIdx.x >> 4) + 16 * k;
            const int col = at_col + ((int)threadIdx.x & 15) * 4;
            v[k] = ns_read4<DTYPE>(m.in, row * m.ld_in + col);
            if (MOMENTUM) old[k] = ns_read4<TFTQ_F32>((const uint8_t *)m.momentum, row * m.ld_momentum + col);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t row = at_row + ((int)threadIdx.x >> 4) + 16 * k;
            const int col = at_col + ((int)threadIdx.x & 15) * 4;
            if (row >= high || col >= wide) continue;
            v[k] = ns_read(m.in, row * m.ld_in + col, DTYPE, wide - col);
            if (MOMENTUM) old[k] = ns_read((const uint8_t *)m.momentum, row * m.ld_momentum + col, TFTQ_F32, wide - col);
        }
    }
    const int parts = (int)ns_parts_of(high, wide);
    double sum = 0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += w.squares[i];
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    const double norm = sqrt(sums[0] + sums[1] + sums[2] + sums[3]);
    const double by = 1.0 / (norm <= (double)p.eps ? (double)p.eps : norm);  // a NaN stays one
    const float scale = ns_scale(norm, p);
    if (piece == 0 && threadIdx.x == 0) *w.scale = scale;
    if (piece == 0)
        for (int i = threadIdx.x; i < NS_SHARED / 2; i += 256) w.tickets[i] = 0;

#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int r = ((int)threadIdx.x >> 4) + 16 * k, c = ((int)threadIdx.x & 15) * 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float u = MOMENTUM ? ns_update(old[k][i], v[k][i], p) : v[k][i];
            const float x = inside || (at_row + r < high && at_col + c + i < wide) ? (float)(u * by) : 0.f;
            if (m.flip) tile[c + i][r] = x;
            else tile[r][c + i] = x;
        }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < 64 * 8; q += 256) {
        const int r = q >> 3, c = (q & 7) * 8;
        ns_h8 hi, lo;
        if (row0 + r < m.rows) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                _Float16 a, b;
                ns_split(tile[r][c + i], scale, &a, &b);
                hi[i] = a, lo[i] = b;
            }
            const int64_t at = ((int64_t)(col0 >> 6) * m.rows + row0 + r) * PANEL_BYTES + c * 2;
            *(ns_h8 *)(w.x + at) = hi;
            *(ns_h8 *)(w.xl + at) = lo;
        }
        if (col0 + r < m.cols) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                _Float16 a, b;
                ns_split(tile[c + i][r], scale, &a, &b);
                hi[i] = a, lo[i] = b;
            }
            const int64_t at = ((int64_t)(row0 >> 6) * m.cols + col0 + r) * PANEL_BYTES + c * 2;
            *(ns_h8 *)(w.t + at) = hi;
            if (precise) *(ns_h8 *)(w.tl + at) = lo;
        }
    }
}

// Where the results go: out = keep out - step X with `update`, else out = X.
struct NsOut {
    uint8_t *out;
    int64_t ld;
    float keep, step;
    int update, dtype;
};
// 8 neighbouring results to the list's matrix: the row, the first column and how many of them exist.
__device__ static __forceinline__ void ns_put(const NsOut &into, int64_t row, int64_t col, int n, const float *v)
{
    const int64_t at = row * into.ld + col;
    const int size = into.dtype == TFTQ_F32 ? 4 : 2;
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
        uint8_t *to = into.out + (at + h) * size;
        tile_f4 o = {v[h], v[h + 1], v[h + 2], v[h + 3]};
        if (n - h <= 0) return;
        if (into.update) {
            const tile_f4 old = ns_read(to, 0, into.dtype, n - h);
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = into.keep * old[i] - into.step * o[i];
        }
        if (n - h >= 4) {
            if (into.dtype == TFTQ_F32) *(ns_f4_any *)to = o;
            else if (into.dtype == TFTQ_F16) *(ns_h4_any *)to = __builtin_convertvector(o, ns_h4_any);
            else *(ns_b4_any *)to = __builtin_convertvector(o, ns_b4_any);
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i >= n - h) continue;
            if (into.dtype == TFTQ_F32) ((float *)to)[i] = o[i];
            else if (into.dtype == TFTQ_F16) ((_Float16 *)to)[i] = (_Float16)o[i];
            else ((__bf16 *)to)[i] = (__bf16)o[i];
        }
    }
}

enum { NS_A, NS_B, NS_X };

// What becomes of a product's sums: E and D, G and F, or X, X^T and the result.  Everything is kept in the
// scale of the fp16 numbers that come of it, so that a value costs a few instructions: a tile's 65 536
// values and their transposes are as much work for the vector units as 20 panels of products are for
// the matrix cores (before: 45).
template <int WHAT, bool PRECISE>
struct NsFinish {
    static constexpr bool LOW = PRECISE || WHAT == NS_X;  // the result's rows have a remainder
    // only what it needs of the matrix, the workspace and the parameters: all of it stays in registers
    NsOut into;
    const uint8_t *old_high, *old_low;
    float *d, *f;
    uint8_t *out, *out_l, *turned, *turned_l;  // panels along the result's rows, and along its columns
    float per_x;                               // one over X's scale, a power of two
    float a, b, c, e, per_ee, aa_to_g, c_to_g, b_to_g, gx_to_x, x_next;
    int r, cols, padded, last, next_last, flip;
    bool mirror;

    __device__ __forceinline__ NsFinish(const NsMatrix &m, const NsParams &p, const NsWork &w, int turn, bool diagonal)
    {
        into.out = m.out, into.ld = m.ld_out, into.keep = p.keep, into.step = m.step, into.update = p.update, into.dtype = p.out_dtype;
        old_high = WHAT == NS_B ? w.e : w.x, old_low = WHAT == NS_B ? w.el : w.xl;
        d = w.d, f = w.f, a = p.a, b = p.b, c = p.c, last = p.last, next_last = p.next_last, flip = m.flip;
        out = WHAT == NS_A ? w.e : WHAT == NS_B ? w.g : w.x, out_l = WHAT == NS_A ? w.el : WHAT == NS_B ? w.gl : w.xl;
        turned = WHAT != NS_X ? out : turn ? w.t : w.t2, turned_l = WHAT != NS_X ? out_l : turn ? w.tl : w.tl2;
        per_x = 1.f / (*w.scale * p.x);
        e = p.e, per_ee = p.per_ee, aa_to_g = p.aa_to_g, c_to_g = p.c_to_g, b_to_g = p.b_to_g, gx_to_x = p.gx_to_x, x_next = p.x_next;
        r = m.rows, cols = WHAT == NS_X ? m.cols : m.rows, padded = (cols + 63) & ~63;
        mirror = WHAT == NS_X ? !last || flip : !diagonal;
    }
    __device__ int64_t at(int i, int j) const { return ((int64_t)(j >> 6) * r + i) * PANEL_BYTES + (j & 63) * 2; }

    // What the results of row i, columns j to j + 7, are made of beside their sums.
    struct Old {
        ns_h8 high, low;
        float di;
    };
    __device__ __forceinline__ Old old(int i, int j) const
    {
        Old o = {};
        if (WHAT == NS_A || i >= r || j >= padded) return o;
        o.high = *(const ns_h8 *)(old_high + at(i, j));
        if (PRECISE || (LOW && !last)) o.low = *(const ns_h8 *)(old_low + at(i, j));
        o.di = WHAT == NS_B ? d[i] : (a + f[i]) * x_next;
        return o;
    }
    // v: the sums of row i, columns j to j + 7, and then their values as numbers (of the last iteration)
    // or in the result's scale.  They go to the rows' panels; `high` and `low` are what is stored there.
    __device__ __forceinline__ void row(int i, int j, float *v, const Old &was, ns_h8 *high, ns_h8 *low) const
    {
        const bool inside = i < r && j < padded;
        if (WHAT == NS_A) {
            if ((unsigned)(i - j) < 8u && i < r) {
#pragma unroll
                for (int n = 0; n < 8; n++)
                    if (i == j + n) d[i] = v[n] * per_x * per_x;
            }
            const float by = per_x * per_x * e;
#pragma unroll
            for (int n = 0; n < 8; n++) v[n] *= by;
        } else if (WHAT == NS_B) {
            if ((unsigned)(i - j) < 8u && i < r) {
#pragma unroll
                for (int n = 0; n < 8; n++)
                    if (i == j + n) f[i] = b * was.di + c * (v[n] * per_ee + was.di * was.di);
            }
            tile_f4 dj[2] = {};
            if (inside) dj[0] = *(const tile_f4 *)(d + j), dj[1] = *(const tile_f4 *)(d + j + 4);
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const float x = PRECISE ? (float)was.high[n] + (float)was.low[n] : (float)was.high[n];
                v[n] = fmaf(x, fmaf(c_to_g, was.di + dj[n / 4][n % 4], b_to_g), v[n] * aa_to_g);
            }
        } else {
#pragma unroll
            for (int n = 0; n < 8; n++) v[n] = fmaf(was.di, (float)was.high[n], fmaf(was.di, (float)was.low[n], v[n] * gx_to_x));
        }
        if (!(i < r && j + 8 <= cols)) {  // zeros past the last row and column
#pragma unroll
            for (int n = 0; n < 8; n++) v[n] = i < r && j + n < cols ? v[n] : 0.f;
        }
        if (WHAT != NS_X && (unsigned)(i - j) < 8u) {  // and on the diagonal
#pragma unroll
            for (int n = 0; n < 8; n++) v[n] = i == j + n ? 0.f : v[n];
        }
        if (WHAT == NS_X && last) {
#pragma unroll
            for (int n = 0; n < 8; n++) v[n] *= per_x;
            if (inside && !flip) ns_put(into, i, j, cols - j, v);
            return;
        }
        split(v, high, low);
        if (!inside) return;
        *(ns_h8 *)(out + at(i, j)) = *high;
        if (PRECISE || (LOW && !next_last)) *(ns_h8 *)(out_l + at(i, j)) = *low;
    }
    __device__ __forceinline__ static void split(const float *v, ns_h8 *high, ns_h8 *low)
    {
        typedef float F2 __attribute__((ext_vector_type(2)));
        typedef _Float16 H2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int n = 0; n < 8; n += 2) {
            const H2 h = __builtin_convertvector(F2{v[n], v[n + 1]}, H2);
            const H2 l = __builtin_convertvector(F2{v[n] - (float)h[0], v[n + 1] - (float)h[1]}, H2);
            (*high)[n] = h[0], (*high)[n + 1] = h[1], (*low)[n] = l[0], (*low)[n + 1] = l[1];
        }
    }
    // Column j, rows i to i + 7, of an iteration that is not the last, to the columns' panels.
    __device__ __forceinline__ void column(int i, int j, const ns_h8 &high, const ns_h8 &low) const
    {
        if (j >= cols || i >= ((r + 63) & ~63)) return;
        const int64_t to = ((int64_t)(i >> 6) * cols + j) * PANEL_BYTES + (i & 63) * 2;
        *(ns_h8 *)(turned + to) = high;
        if (PRECISE) *(ns_h8 *)(turned_l + to) = low;
    }
    // The last one's values of column j, rows i to i + 7.
    __device__ __forceinline__ void column_out(int i, int j, const float *v) const
    {
        if (j < cols && i < r) ns_put(into, j, i, r - i, v);
    }
};

// How many tiles of `size` rows cover n of them and what fills the last panel up, whose zeros they write.
__host__ __device__ static inline int ns_tiles(int n, int size) { return (((n + 63) & ~63) + size - 1) / size; }

// What a product contracts, and the tile of a matrix that piece `piece` is.
template <int WHAT>
struct NsProduct {
    const uint8_t *ah, *al, *bh, *bl;
    int a_rows, b_rows, panels;
    // part `split` of `splits` of the panels
    __device__ __forceinline__ NsProduct(const NsMatrix &m, const NsWork &w, int turn, int split, int splits)
    {
        ah = WHAT == NS_A ? w.x : WHAT == NS_B ? w.e : w.g, al = WHAT == NS_A ? w.xl : WHAT == NS_B ? w.el : w.gl;
        bh = WHAT == NS_A ? w.x : WHAT == NS_B ? w.e : turn ? w.t2 : w.t, bl = WHAT == NS_A ? w.xl : WHAT == NS_B ? w.el : turn ? w.tl2 : w.tl;
        a_rows = m.rows, b_rows = WHAT == NS_X ? m.cols : m.rows;
        panels = ((WHAT == NS_A ? m.cols : m.rows) + 63) >> 6;
        if (splits > 1) {
            const int first = panels * split / splits;
            panels = panels * (split + 1) / splits - first;
            const int64_t a = (int64_t)first * a_rows * PANEL_BYTES, b = (int64_t)first * b_rows * PANEL_BYTES;
            ah += a, al += a, bh += b, bl += b;
        }
    }
    __device__ __forceinline__ void tile(int piece, int high, int wide, int *tm, int *tn) const
    {
        if (WHAT == NS_X) {
            tile_place(piece, ns_tiles(a_rows, high), ns_tiles(b_rows, wide), tm, tn);
            return;
        }
        int n = (int)((sqrtf(8.f * piece + 1.f) - 1.f) * 0.5f);  // column n of the upper triangle has n + 1 tiles
        while ((n + 1) * (n + 2) / 2 <= piece) n++;
        while (n * (n + 1) / 2 > piece) n--;
        *tn = n, *tm = piece - n * (n + 1) / 2;
    }
};

// Column lane % 16, rows 8 (lane / 16) to + 7, of 32 rows of 16 numbers in LDS.  Of ds_read_b64_tr_b16 every 16
// lanes name 4 rows of 16 numbers, 4 of them each, and get a column's 4 each.
__device__ static inline ns_h8 ns_down(const _Float16 *from, int pitch, int lane)
{
    typedef short S4 __attribute__((ext_vector_type(4)));
    typedef _Float16 H4 __attribute__((ext_vector_type(4)));
    const _Float16 *at = from + ((lane >> 4) * 8 + (lane & 15) / 4) * pitch + (lane & 3) * 4;
    const H4 a = __builtin_bit_cast(H4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4 *)at));
    const H4 b = __builtin_bit_cast(H4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4 *)(at + 4 * pitch)));
    return ns_h8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Where tiles are fewer than compute units, workgroups share one, each a part of its panels: every one
// stores its sums, and the last one to be done adds all of them up, in their order, and goes on alone.
// take(i): the i-th vector of the thread's sums, put(i, v): it becomes v.
struct NsSplit {
    int tile, split, splits;
    __device__ __forceinline__ NsSplit(const NsMatrix &m, int piece, bool shared)
    {
        tile = piece, split = 0, splits = 1;
        if (!shared || m.splits == 1) return;
        const int tiles = m.pieces / m.splits;  // a part of all tiles, then the next part
        split = piece / tiles, tile = piece - split * tiles, splits = m.splits;
    }
    // The sums are stored and loaded at the device's scope, past the caches of one XCD, and a workgroup takes
    // its ticket when all of its stores are done: no cache has to be written back or emptied (with
    // fences that do so, 70 us a launch of 500 workgroups).
    template <int VECTORS, int THREADS, class A, class B>
    __device__ __forceinline__ bool join(const NsWork &w, int *last, A take, B put) const
    {
        uint64_t *sums = (uint64_t *)w.sums + (int64_t)tile * splits * VECTORS * THREADS * 2 + threadIdx.x;
        if (threadIdx.x < THREADS) {
#pragma unroll
            for (int i = 0; i < VECTORS; i++) {
                const tile_f4 v = take(i);
                uint64_t *at = sums + (split * VECTORS + i) * THREADS * 2;
                __hip_atomic_store(at, pair(v[0], v[1]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(at + THREADS, pair(v[2], v[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            *last = __hip_atomic_fetch_add(w.tickets + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == splits - 1;
            if (*last) __hip_atomic_store(w.tickets + tile, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
        }
        __syncthreads();
        if (!*last) return false;
        if (threadIdx.x < THREADS) {
            tile_f4 v[VECTORS] = {};
            for (int n = 0; n < splits; n++) {
#pragma unroll
                for (int i = 0; i < VECTORS; i++) {
                    const uint64_t *at = sums + (n * VECTORS + i) * THREADS * 2;
                    const uint64_t x = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    const uint64_t y = __hip_atomic_load(at + THREADS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    v[i] += tile_f4{__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32)), __uint_as_float((uint32_t)y), __uint_as_float((uint32_t)(y >> 32))};
                }
            }
#pragma unroll
            for (int i = 0; i < VECTORS; i++) put(i, v[i]);
        }
        return true;
    }
    __device__ __forceinline__ static uint64_t pair(float a, float b) { return __float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32; }
};

// LDS of a product's workgroup: the tile's buffers, and when they are done with its strips as sums and as
// two fp16 numbers each.
template <class T>
struct NsLds {
    static constexpr int STRIPS = T::WAVES * (32 * T::PITCH * 4 + 2 * 32 * (T::WN + 8) * 2);
    static constexpr int BYTES = T::LDS > STRIPS ? T::LDS : STRIPS;
};

// One of the products, a tile per workgroup.  4096x14336 with one product each (us, and the rate of the
// work that symmetry leaves): A 255 (0.94 PFLOP/s), B 82 (0.84), X 552 (0.87; a loop without an end
// 1.23): X moves 10 bytes an element besides, with nothing to multiply meanwhile.  SHARED: some tiles have
// several workgroups (NsSplit).
template <class T, int WHAT, bool PRECISE, bool SHARED>
__global__ __launch_bounds__(T::THREADS) void k_ns_product(int count, int turn, const NsLaunch l, const NsParams p)
{
    __shared__ __attribute__((aligned(128))) uint8_t lds[NsLds<T>::BYTES];
    int matrix, piece, tm, tn;
    if (!ns_tile(l, count, blockIdx.x, &matrix, &piece)) return;
    const NsMatrix m = l.m[matrix];
    const NsWork w = ns_work(m.work, m.rows, m.cols, m.flip, PRECISE);
    const NsSplit mine(m, piece, SHARED);
    const NsProduct<WHAT> o(m, w, turn, mine.split, mine.splits);
    o.tile(mine.tile, T::ROWS, T::COLS, &tm, &tn);
    const int row0 = tm * T::ROWS, col0 = tn * T::COLS;
    T t;
    auto place = [&](int, int *r0, int *c0) { *r0 = row0, *c0 = col0; };
    auto done = [](int, int) {};
    if constexpr (PRECISE) t.multiply(TileTriple{{o.ah, o.al, o.bh, o.bl, o.a_rows, o.b_rows, o.panels}}, 3 * o.panels, 1, place, lds, done);
    else t.multiply(TilePair{{o.ah, nullptr, o.a_rows}, {o.bh, nullptr, o.b_rows}}, o.panels, 1, place, lds, done);
    if constexpr (SHARED) {
        if (mine.splits > 1) {
            static_assert(T::TM == 1 && T::TN == 1, "");
            if (!mine.template join<4, T::THREADS>(w, (int *)lds, [&](int i) {
                    return tile_f4{t.acc[0][0][4 * i], t.acc[0][0][4 * i + 1], t.acc[0][0][4 * i + 2], t.acc[0][0][4 * i + 3]};
                }, [&](int i, tile_f4 v) {
#pragma unroll
                    for (int n = 0; n < 4; n++) t.acc[0][0][4 * i + n] = v[n];
                }))
                return;
            __syncthreads();  // `last` has been read: the strips may take its place
        }
    }

    const NsFinish<WHAT, PRECISE> finish(m, p, w, turn, tm == tn);
    constexpr int ACROSS = T::WN / 8, PASSES = 32 * ACROSS / 64;  // 8 neighbours of a row per lane
    static_assert(32 * ACROSS % 64 == 0 && T::WN % 16 == 0, "");
    // the fp16 numbers of a strip, behind the strips themselves
    constexpr int PITCH16 = T::WN + 8, HALF = 32 * PITCH16;
    static_assert(T::WAVES * (32 * T::PITCH * 4 + 2 * HALF * 2) <= NsLds<T>::BYTES, "");
    const int lane = threadIdx.x & 63;
    _Float16 *halves = (_Float16 *)(lds + T::WAVES * 32 * T::PITCH * 4) + tile_wave() * 2 * HALF;
    typename NsFinish<WHAT, PRECISE>::Old was[2][PASSES];  // of the next strip while one is finished
    const std::make_integer_sequence<int, PASSES> passes;
    t.store_strips(row0, col0, lds, [&](auto i, int row, int col) __attribute__((always_inline)) {
        tile_each(passes, [&](auto q) __attribute__((always_inline)) {
            was[i & 1][q] = finish.old(row + (lane + 64 * q) / ACROSS, col + (lane + 64 * q) % ACROSS * 8);
        });
    }, [&](auto i, float *strip, int row, int col) __attribute__((always_inline)) {
        const bool last = WHAT == NS_X && finish.last;
        tile_each(passes, [&](auto q) __attribute__((always_inline)) {
            const int at = (lane + 64 * q) / ACROSS, c = (lane + 64 * q) % ACROSS * 8;
            float v[8];
            tile_f4 *from = (tile_f4 *)__builtin_assume_aligned(strip + at * T::PITCH + c, 16);
            *(tile_f4 *)v = from[0], *(tile_f4 *)(v + 4) = from[1];
            ns_h8 high, low;
            finish.row(row + at, col + c, v, was[i & 1][q], &high, &low);
            if (!finish.mirror) return;
            if (last) {
                from[0] = *(tile_f4 *)v, from[1] = *(tile_f4 *)(v + 4);
            } else {
                *(ns_h8 *)__builtin_assume_aligned(halves + at * PITCH16 + c, 16) = high;
                if (PRECISE) *(ns_h8 *)__builtin_assume_aligned(halves + HALF + at * PITCH16 + c, 16) = low;
            }
        });
        T::wave_fence();
        if (!finish.mirror) return;
        if (last) {
#pragma unroll 1
            for (int q = lane; q < T::WN * 4; q += 64) {  // 8 rows of a column per lane
                float v[8];
#pragma unroll
                for (int n = 0; n < 8; n++) v[n] = strip[((q & 3) * 8 + n) * T::PITCH + (q >> 2)];
                finish.column_out(row + (q & 3) * 8, col + (q >> 2), v);
            }
            return;
        }
#pragma unroll
        for (int c = 0; c < T::WN; c += 16) {  // 8 rows of 16 columns per 16 lanes
            ns_h8 high = ns_down(halves + c, PITCH16, lane), low = high;
            if (PRECISE) low = ns_down(halves + HALF + c, PITCH16, lane);
            finish.column(row + (lane >> 4) * 8, col + c + (lane & 15), high, low);
        }
    });
}

// The same for matrices of few tiles, where a kernel's time is that of the loads it waits for: a tile of
// 32 x 32 per workgroup, whose 8 wavefronts share the panels between them, take their operands straight
// from memory with all of a panel's loads in flight, and add up in LDS.  256x512 with three products: A 7.2,
// B 6.6, X 5.9 us, of which a launch and the ways to memory and back are nearly all.
template <int WHAT, bool PRECISE, bool SHARED>
__global__ __launch_bounds__(512) void k_ns_small(int count, int turn, const NsLaunch l, const NsParams p)
{
    constexpr int WAVES = 8, PITCH = 36;
    __shared__ __attribute__((aligned(128))) float sums[WAVES][32 * PITCH];
    __shared__ int last;
    int matrix, piece, tm, tn;
    if (!ns_tile(l, count, blockIdx.x, &matrix, &piece)) return;
    const NsMatrix m = l.m[matrix];
    const NsWork w = ns_work(m.work, m.rows, m.cols, m.flip, PRECISE);
    const NsSplit mine(m, piece, SHARED);
    const NsProduct<WHAT> o(m, w, turn, mine.split, mine.splits);
    o.tile(mine.tile, 32, 32, &tm, &tn);
    const int lane = threadIdx.x & 63, wave = tile_wave(), half = lane >> 5;
    const int64_t a_at = (int64_t)min(tm * 32 + (lane & 31), o.a_rows - 1) * PANEL_BYTES + half * 16;
    const int64_t b_at = (int64_t)min(tn * 32 + (lane & 31), o.b_rows - 1) * PANEL_BYTES + half * 16;
    tile_f16 acc = {};
    for (int s = wave; s < o.panels; s += WAVES) {
        const int64_t a = a_at + (int64_t)s * o.a_rows * PANEL_BYTES, b = b_at + (int64_t)s * o.b_rows * PANEL_BYTES;
        tile_h8 ah[4], bh[4], al[4], bl[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            ah[q] = *(const tile_h8 *)(o.ah + a + q * 32), bh[q] = *(const tile_h8 *)(o.bh + b + q * 32);
            if (PRECISE) al[q] = *(const tile_h8 *)(o.al + a + q * 32), bl[q] = *(const tile_h8 *)(o.bl + b + q * 32);
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {  // b first: a lane's sums are neighbours in a row (tftq_tile.h)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[q], ah[q], acc, 0, 0, 0);
            if (PRECISE) {
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[q], al[q], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(bl[q], ah[q], acc, 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < 4; g++)
        *(tile_f4 *)(sums[wave] + (lane & 31) * PITCH + 8 * g + 4 * half) = tile_f4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};

    const NsFinish<WHAT, PRECISE> finish(m, p, w, turn, tm == tn);
    const int id = threadIdx.x, at = id >> 2, c = (id & 3) * 8;  // the first 128 threads
    typename NsFinish<WHAT, PRECISE>::Old was = {};
    if (id < 128) was = finish.old(tm * 32 + at, tn * 32 + c);
    __syncthreads();
    float v[8];
    if (id < 128) {
#pragma unroll
        for (int n = 0; n < 8; n++) {
            v[n] = sums[0][at * PITCH + c + n];
#pragma unroll
            for (int k = 1; k < WAVES; k++) v[n] += sums[k][at * PITCH + c + n];
        }
    }
    if (SHARED && mine.splits > 1 && !mine.template join<2, 128>(w, &last, [&](int i) { return tile_f4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]}; },
                                                    [&](int i, tile_f4 to) { v[4 * i] = to[0], v[4 * i + 1] = to[1], v[4 * i + 2] = to[2], v[4 * i + 3] = to[3]; }))
        return;
    if (id < 128) {
        ns_h8 high, low;
        finish.row(tm * 32 + at, tn * 32 + c, v, was, &high, &low);
#pragma unroll
        for (int n = 0; n < 8; n++) sums[0][at * PITCH + c + n] = v[n];
    }
    if (!finish.mirror) return;
    __syncthreads();
    if (id < 128) {
        const int j = id >> 2, i = (id & 3) * 8;
        float v[8];
#pragma unroll
        for (int n = 0; n < 8; n++) v[n] = sums[0][(i + n) * PITCH + j];
        if (WHAT == NS_X && finish.last) {
            finish.column_out(tm * 32 + i, tn * 32 + j, v);
        } else {
            ns_h8 high, low;
            finish.split(v, &high, &low);
            finish.column(tm * 32 + i, tn * 32 + j, high, low);
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <class F>
static int launch_over(NsLaunch &l, F workgroups, bool eighths, const void *kernel, int threads, const NsParams &p, int extra, hipStream_t st)
{
    int64_t total = 0;
    for (int i = 0; i < l.count; i++) {
        const int64_t n = workgroups(l.m[i]) * l.m[i].splits;
        l.first[i] = (int)total, l.m[i].pieces = (int)n;
        total += eighths ? (n + 7) / 8 : n;
    }
    for (int i = l.count; i < NS_MOST; i++) l.first[i] = INT_MAX;
    void *args[] = {(void *)&l.count, (void *)&extra, (void *)&l, (void *)&p};
    return (int)hipLaunchKernel(kernel, dim3((unsigned)(eighths ? total * 8 : total)), dim3(threads), args, 0, st);
}

static int64_t tiles(const NsMatrix &m, int what, int high, int wide)
{
    const int64_t r = ns_tiles(m.rows, high), k = ns_tiles(m.cols, wide);
    return what == NS_X ? r * k : r * (r + 1) / 2;
}

static bool ns_shared(const NsLaunch &l)
{
    return std::any_of(l.m, l.m + l.count, [](const NsMatrix &m) { return m.splits > 1; });
}

template <class T, int WHAT>
static int launch_tiles(NsLaunch &l, bool precise, const NsParams &p, int turn, hipStream_t st)
{
    const void *k = precise ? (const void *)k_ns_product<T, WHAT, true, false> : (const void *)k_ns_product<T, WHAT, false, false>;
    if constexpr (T::ROWS == 64) {
        if (ns_shared(l)) k = precise ? (const void *)k_ns_product<T, WHAT, true, true> : (const void *)k_ns_product<T, WHAT, false, true>;
    }
    return launch_over(l, [](const NsMatrix &m) { return tiles(m, WHAT, T::ROWS, T::COLS); }, true, k, T::THREADS, p, turn, st);
}

// How many workgroups share a tile of `all` in a launch, each at least `least` of its panels: a panel for every
// wavefront of k_ns_small; what outweighs the sums' way through memory, 3 us, in tiles of 64 x 64.  No more
// than 16, whose sums one workgroup adds up.  Graph replays of the whole orthogonalisation, us, with a
// workgroup to a tile and so: fp32 64x3584 195, 102; 64x16384 666, 148; 256x16384 740, 283; 1024x16384 1840,
// 1261; 768x1024 262, 239; 1024x1024 287, 291; bf16 256x16384 403, 194; 1024x16384 710, 547 (from 8 panels on
// 1024x1024 bf16 is shared too: 151, 192).
static int ns_splits(int64_t all, int64_t panels, int least)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>({NS_SHARED / std::max<int64_t>(all, 1), panels / least, 16}));
}
static int64_t ns_panels(const NsMatrix &m, int what) { return ((what == NS_A ? m.cols : m.rows) + 63) / 64; }
static int ns_least(int size, bool precise) { return size == 32 ? 8 : precise ? 6 : 16; }
static int64_t ns_all(const NsLaunch &l, int what, int high, int wide)
{
    int64_t all = 0;
    for (int i = 0; i < l.count; i++) all += tiles(l.m[i], what, high, wide);
    return all;
}

// About how long a product of the matrices of a launch takes in tiles of a size.
static double ns_time(const NsLaunch &l, int what, const TileShape &t, bool precise)
{
    double work = 0, longest = 0, count = 0, more = 0;
    const int64_t all = ns_all(l, what, t.high, t.wide);
    for (int i = 0; i < l.count; i++) {
        const double n = (double)tiles(l.m[i], what, t.high, t.wide), panels = (double)ns_panels(l.m[i], what) * (precise ? 3 : 1);
        const int splits = t.high == 64 ? ns_splits(all, ns_panels(l.m[i], what), ns_least(64, precise)) : 1;
        count += n * splits, work += n * panels, longest = std::max(longest, panels / splits);
        if (splits > 1) more = 12 * t.one;  // the sums' way through memory
    }
    return tile_time(t, count, work, longest) + more;
}

// The same for k_ns_small, to which one panel of its 8 wavefronts after the other comes from memory, on every
// unit that has a workgroup at once, and beside whose launch that of a tile kernel takes 0.5 more.  Nothing
// is faster where there is one such panel.  From (us) fp32 256x512, A (1 panel, 36 tiles) 7.4; 870x6665, A (14 panels, 406 tiles) 108, B (2, 406) 17.
static double ns_small_time(const NsLaunch &l, int what, bool precise)
{
    const int64_t all = ns_all(l, what, 32, 32);
    int64_t count = 0, panels = 0;
    double more = -0.5;
    for (int i = 0; i < l.count; i++) {
        const int splits = ns_splits(all, ns_panels(l.m[i], what), ns_least(32, precise));
        count += tiles(l.m[i], what, 32, 32) * splits, panels = std::max(panels, (ns_panels(l.m[i], what) + 8 * splits - 1) / (8 * splits));
        if (splits > 1) more = 0.7;
    }
    panels *= (count + 255) / 256;
    return panels <= 1 ? 0 : 2.2 + (precise ? 2.1 : 0.9) * (double)panels + more;
}

// One of the three products for all matrices of a launch.  k_ns_small and tiles of 64 x 64, graph replays of the
// whole orthogonalisation, us: fp32 512x512 130, 183; 512x768 159, 191; 768x1024 282, 239; 1024x1024 432,
// 291.  bf16 512x512 92, 105; 512x768 107, 112; 640x640 119, 121; 768x1024 181, 142.
template <int WHAT>
static int product(NsLaunch &l, bool precise, const NsParams &p, int turn, hipStream_t st)
{
    // the matrices with most panels first: the last workgroups are then short ones
    std::stable_sort(l.m, l.m + l.count, [](const NsMatrix &x, const NsMatrix &y) { return ns_panels(x, WHAT) > ns_panels(y, WHAT); });
    auto share = [&](int size) {
        const int64_t all = ns_all(l, WHAT, size, size);
        for (int i = 0; i < l.count; i++) l.m[i].splits = size > 64 ? 1 : ns_splits(all, ns_panels(l.m[i], WHAT), ns_least(size, precise));
    };
    const TileShape choice[] = {TILES_256, WHAT == NS_X ? TILES_192X256 : TILES_192, TILES_128, TILES_64};
    int best = 0;
    for (int i = 1; i < 4; i++)
        if (ns_time(l, WHAT, choice[i], precise) < ns_time(l, WHAT, choice[best], precise)) best = i;
    if (ns_small_time(l, WHAT, precise) < ns_time(l, WHAT, choice[best], precise)) {
        share(32);
        const void *k = ns_shared(l) ? precise ? (const void *)k_ns_small<WHAT, true, true> : (const void *)k_ns_small<WHAT, false, true>
                        : precise ? (const void *)k_ns_small<WHAT, true, false> : (const void *)k_ns_small<WHAT, false, false>;
        return launch_over(l, [](const NsMatrix &m) { return tiles(m, WHAT, 32, 32); }, true, k, 512, p, turn, st);
    }
    share(choice[best].high);
    switch (best) {
    case 0: return launch_tiles<Tile<256, 256, 2, 4, false>, WHAT>(l, precise, p, turn, st);
    case 1:
        if (WHAT == NS_X) return launch_tiles<Tile<192, 256, 2, 4, false>, NS_X>(l, precise, p, turn, st);
        return launch_tiles<Tile<192, 192, 2, 2, false>, WHAT == NS_X ? NS_A : WHAT>(l, precise, p, turn, st);
    case 2: return launch_tiles<Tile<128, 128, 2, 2, false>, WHAT>(l, precise, p, turn, st);
    default: return launch_tiles<Tile<64, 64, 2, 2, false, 3>, WHAT>(l, precise, p, turn, st);
    }
}

// Bytes of workspace of a matrix: its parts and, for the most workgroups that may ever share its tiles (those
// of a launch of its own), their sums.
static int64_t ns_bytes(int64_t r, int64_t k, bool flip, bool precise)
{
    NsMatrix m = {};
    m.rows = (int)r, m.cols = (int)k;
    int64_t sums = 0;
    for (int what = NS_A; what <= NS_X; what++)
        for (int size = 32; size <= 64; size += 32) {
            const int64_t all = tiles(m, what, size, size);
            const int splits = ns_splits(all, ns_panels(m, what), ns_least(size, precise));
            if (splits > 1) sums = std::max(sums, all * splits * size * size * 4);
        }
    return ns_work(nullptr, r, k, flip, precise).bytes + sums;
}

static bool ns_shapes_ok(int n, const int64_t *shapes)
{
    for (int i = 0; i < 2 * n; i++)
        if (shapes[i] < 0 || shapes[i] > NS_LONGEST) return false;
    return true;
}

// Whether a matrix of r rows (columns, if these are fewer) takes three products.  The errors of the one of 11
// bits are those of many roundings, and average, the better the larger r is.  They are largest where one direction
// holds the norm: what rounds off it is multiplied by up to 480 in the others.  Rank one with noise of 0 to 1e-3, bf16
// results, worst of 24 (the same rounded once 1.7e-3, at most 3.9e-3): r = 64 1.1e-2, 96 7.8e-3, 128 6.7e-3, 160 5.0e-3,
// 192 3.6e-3, 224 4.1e-3, 256 3.0e-3, 512 2.3e-3.  A matrix of fewer than 192 rows is at most three tiles high, and its products
// wait for memory more than for the matrix cores: one and three products, us, 64x512 67, 84; 128x1024 83, 100;
// 160x5120 115, 141; 24 of 128x256 108, 141; 24 of 128x2048 217, 258 (256x2048 102, 131; 512x4096 153, 235).
static bool ns_precise(int64_t r, int precise) { return precise || r < 192; }

// Whether the matrices of one product are so few and small that they join those of three in their launches: two
// times their work more, but no 17 launches of their own (bf16, us, together and apart: 322x322 with 1x322 and
// 322x1 112, 148; 640x640 with 512x1 184, 183; four of 256x1024 with 128x1024 175, 213; ten of 844x211 with two of
// 211x1 218, 226; three of 512x512 with three of 128x512 201, 232; four of 300x1200 with 1x300 187, 202; 768x768
// with four of 96x768 237, 253; above the limit 1024x1024 with 1024x1 286, 230, two of 1024x1024 with two of
// 128x1024 379, 293).
static bool ns_together(int n, const int64_t *shapes)
{
    double work = 0;
    bool narrow = false;
    for (int i = 0; i < n; i++) {
        const double a = (double)shapes[2 * i], b = (double)shapes[2 * i + 1], r = std::min(a, b);
        if (r > 0 && ns_precise((int64_t)r, 0)) narrow = true;
        else work += r * a * b;
    }
    return narrow && n <= NS_MOST && work <= 5e8;
}

// Squares of 64 of a launch's matrices: no kernel has more workgroups of 256 threads, or half as many of
// 512, and a launch has fewer than 2^32 threads.
constexpr int64_t NS_SQUARES = 1 << 23;

// f(the matrices of one launch, how many, whether they take three products, bytes of workspace) for the whole list.
template <class F>
static int ns_parts(int n, const int64_t *shapes, int precise, F f)
{
    if (!precise && ns_together(n, shapes)) precise = 1;
    for (int kind = 0; kind < 2; kind++) {
        int at[NS_MOST], count = 0;
        int64_t bytes = 0, squares = 0;
        for (int i = 0; i < n; i++) {
            const int64_t a = shapes[2 * i], b = shapes[2 * i + 1], r = a < b ? a : b;
            if (r == 0 || ns_precise(r, precise) != (kind != 0)) continue;
            const int64_t more = ((a + 63) / 64) * ((b + 63) / 64);
            if (more > NS_SQUARES) return TFTQ_E_SHAPE;
            if (count == NS_MOST || squares + more > NS_SQUARES) {
                if (const int rc = f(at, count, kind != 0, bytes)) return rc;
                count = 0, bytes = 0, squares = 0;
            }
            bytes += ns_bytes(r, a < b ? b : a, a > b, kind != 0);
            squares += more;
            at[count++] = i;
        }
        if (count)
            if (const int rc = f(at, count, kind != 0, bytes)) return rc;
    }
    return 0;
}

extern "C" int64_t tftq_newton_schulz_workspace(int n, const int64_t *shapes, int precise)
{
    if (n < 0 || (n > 0 && !shapes)) return TFTQ_E_ARG;
    if (!ns_shapes_ok(n, shapes)) return TFTQ_E_SHAPE;
    int64_t most = 0;
    const int rc = ns_parts(n, shapes, precise, [&](const int *, int, bool, int64_t bytes) {
        most = std::max(most, bytes);
        return 0;
    });
    return rc ? rc : most;
}

template <int DTYPE>
static const void *ns_first(bool momentum) { return momentum ? (const void *)k_ns_squares<DTYPE, true> : (const void *)k_ns_squares<DTYPE, false>; }
template <int DTYPE>
static const void *ns_second(bool momentum) { return momentum ? (const void *)k_ns_start<DTYPE, true> : (const void *)k_ns_start<DTYPE, false>; }

// The scales of every iteration, powers of two.  X starts with singular values of at most 1 (its norm); an iteration
// takes each of them, x, to a x + b x^3 + c x^5, and A and B have eigenvalues x^2 and b x^2 + c x^4: what these
// are at most over all x up to the last bound is the next one, and bounds the matrices' elements.  Half of fp16's range
// is left for rounding.  The scales end at 2^-50, for X of 4e9.
struct NsScales {
    double bound = 1;
    static float fit(float most, double bound)
    {
        while (bound * 2 * most > 65504. && most > 0x1p-50f) most *= 0.5f;
        return most;
    }
    // the largest of |f| at 0, at `end` and at the given ones of its extrema that lie between
    template <class F>
    static double largest(F f, double end, std::initializer_list<double> extrema)
    {
        double most = fabs(f(end));
        for (double at : extrema)
            if (at > 0 && at < end) most = std::max(most, fabs(f(at)));
        return most;
    }
    // p's scales for its coefficients
    void next(NsParams &p)
    {
        const double a = p.a, b = p.b, c = p.c, square = bound * bound;
        const float x = fit(SCALE_X, bound), e = fit(SCALE_E, square);
        const float g = fit(SCALE_G, largest([&](double y) { return b * y + c * y * y; }, square, {-b / (2 * c)}));
        // extrema of a x + b x^3 + c x^5: a + 3 b y + 5 c y^2 = 0 with y = x^2
        const double root = sqrt(9 * b * b - 20 * a * c);
        bound = largest([&](double x) { return x * (a + x * x * (b + c * x * x)); }, bound,
                        {sqrt((-3 * b + root) / (10 * c)), sqrt((-3 * b - root) / (10 * c)), sqrt(-a / (3 * b))});
        p.x = x / SCALE_X, p.x_next = p.last ? 1.f : fit(SCALE_X, bound) / x;
        p.e = e, p.per_ee = 1.f / (e * e);
        p.aa_to_g = p.c * (g / (e * e)), p.c_to_g = p.c * (g / e), p.b_to_g = p.b * (g / e);
        p.gx_to_x = p.x_next / g;
    }
};

static bool ns_dtype_ok(int d) { return d == TFTQ_F32 || d == TFTQ_F16 || d == TFTQ_BF16; }

extern "C" int tftq_newton_schulz(const tftq_ns *what, void *workspace, int64_t workspace_bytes, int device, void *stream)
{
    if (!what || what->n < 0) return TFTQ_E_ARG;
    const tftq_ns &s = *what;
    if (s.n == 0) return 0;
    if (!s.shapes || !s.in || !s.in_stride || !s.out || !s.out_stride || !s.coefficients || s.iterations < 1) return TFTQ_E_ARG;
    if ((s.momenta != nullptr) != (s.momenta_stride != nullptr)) return TFTQ_E_ARG;
    if (!ns_dtype_ok(s.in_dtype) || !ns_dtype_ok(s.out_dtype)) return TFTQ_E_DTYPE;
    if (!ns_shapes_ok(s.n, s.shapes)) return TFTQ_E_SHAPE;
    for (int i = 0; i < s.n; i++) {
        const int64_t rows = s.shapes[2 * i], cols = s.shapes[2 * i + 1], least = rows > 1 ? cols : 0;
        if (rows == 0 || cols == 0) continue;
        if (!s.in[i] || !s.out[i] || s.in_stride[i] < least || s.out_stride[i] < least) return TFTQ_E_ARG;
        if (s.momenta && (!s.momenta[i] || s.momenta_stride[i] < least)) return TFTQ_E_ARG;
    }
    const int64_t needed = tftq_newton_schulz_workspace(s.n, s.shapes, s.precise);
    if (needed <= 0) return (int)needed;
    if (workspace_bytes < needed) return TFTQ_E_SIZE;
    if (!workspace || ((uintptr_t)workspace & 127)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    hipStream_t st = (hipStream_t)stream;

    return ns_parts(s.n, s.shapes, s.precise, [&](const int *at, int count, bool precise, int64_t) {
        NsLaunch l;
        l.count = 0;
        uint8_t *work = (uint8_t *)workspace;
        for (int q = 0; q < count; q++) {
            const int i = at[q];
            const int64_t rows = s.shapes[2 * i], cols = s.shapes[2 * i + 1];
            NsMatrix &m = l.m[l.count++];
            m.in = (const uint8_t *)s.in[i], m.out = (uint8_t *)s.out[i], m.momentum = s.momenta ? s.momenta[i] : nullptr;
            m.ld_in = s.in_stride[i], m.ld_out = s.out_stride[i], m.ld_momentum = s.momenta ? s.momenta_stride[i] : 0;
            m.flip = rows > cols;
            m.rows = (int)std::min(rows, cols), m.cols = (int)std::max(rows, cols);
            m.step = s.steps ? s.steps[i] : 0.f;
            m.work = work;
            m.splits = 1;
            work += ns_bytes(m.rows, m.cols, m.flip, precise);
        }
        float growth = 1.f;
        for (int it = 0; it < s.iterations; it++) growth *= fmaxf(1.f, fabsf(s.coefficients[3 * it]));
        NsParams p = {s.momentum, s.keep, 0, 0, 0, s.eps, growth, s.nesterov, s.out_dtype, s.steps != nullptr};
        NsScales scales;
        const bool with = s.momenta != nullptr;
        const void *squares, *start;
        switch (s.in_dtype) {
        case TFTQ_F32: squares = ns_first<TFTQ_F32>(with), start = ns_second<TFTQ_F32>(with); break;
        case TFTQ_F16: squares = ns_first<TFTQ_F16>(with), start = ns_second<TFTQ_F16>(with); break;
        default: squares = ns_first<TFTQ_BF16>(with), start = ns_second<TFTQ_BF16>(with); break;
        }
        int rc = launch_over(l, [](const NsMatrix &m) {
            const int64_t high = m.flip ? m.cols : m.rows, wide = m.flip ? m.rows : m.cols;
            return ns_parts_of(high, wide);
        }, false, squares, 256, p, precise, st);
        if (rc) return rc;
        rc = launch_over(l, [](const NsMatrix &m) { return (int64_t)((m.rows + 63) / 64) * ((m.cols + 63) / 64); }, false, start, 256,
                         p, precise, st);
        if (rc) return rc;
        for (int it = 0; it < s.iterations; it++) {
            p.a = s.coefficients[3 * it], p.b = s.coefficients[3 * it + 1], p.c = s.coefficients[3 * it + 2];
            p.last = it + 1 == s.iterations, p.next_last = it + 2 == s.iterations;
            scales.next(p);
            if ((rc = product<NS_A>(l, precise, p, it & 1, st)) || (rc = product<NS_B>(l, precise, p, it & 1, st)) ||
                (rc = product<NS_X>(l, precise, p, it & 1, st)))
                return rc;
        }
        return 0;
    });
}
