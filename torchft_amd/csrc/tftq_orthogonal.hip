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
// leave out and the term (a + F) X takes in.  Relative error of the result against 64 bits, one
// product each, matrices of 64x64 to 1024x1024 with even, low-rank and 1/i spectra: 2.4e-4 to 1.3e-3
// (bf16 results are rounded by 1.7e-3; A, B and X in plain bf16: 1.3e-2 to 7.7e-2, in plain fp16 up to
// 9e-3).  `precise`: A, B and X^T have second numbers too and every product is three, high x high +
// low x high + high x low: 5e-7 to 5e-6, where fp32 products give 1e-6 to 6e-6, at three times the work
// of the 16-bit cores, which is a fifth of what the fp32 ones would take.
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and stored twice.
// X^T is stored beside X so that all three products contract rows of both operands (tftq_tile.h).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "tftq_device.h"
#include "tftq_tile.h"

typedef _Float16 ns_h8 __attribute__((ext_vector_type(8)));

constexpr int NS_MOST = 24;            // matrices of a launch: their descriptors travel in its arguments
constexpr int64_t NS_LONGEST = 1 << 24;  // rows or columns
// |X| <= ~1.2, |A| <= ~1.5, |B| <= ~3 with the usual coefficients; others may pass these a few times over.
// X of a gradient so small that eps divides it stays small: its scale is larger by a power of two (ns_scale).
constexpr float SCALE_X = 16384.f, SCALE_E = 4096.f, SCALE_G = 2048.f;
constexpr int NORM_ROWS = 64, NORM_COLS = 1024;  // of the matrix as it lies: the part that a workgroup sums the squares of

struct NsMatrix {
    const uint8_t *in;
    float *momentum;
    uint8_t *out;
    int64_t ld_in, ld_momentum, ld_out;
    uint8_t *work;
    int rows, cols;  // of X
    int flip;        // X is the transpose of the matrix as it lies
    int whole_out;   // vectors of out's rows are aligned
    float step;      // out = keep * out - step * X with NsParams::update, else out = X
    int first;       // the launch's first workgroup of this matrix
};
struct NsLaunch {
    int count;
    NsMatrix m[NS_MOST];
};
struct NsParams {
    float momentum, keep, a, b, c, eps, growth;
    int nesterov, in_dtype, out_dtype, update, last;
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
    int64_t bytes;
};
__host__ __device__ static inline NsWork ns_work(uint8_t *base, int64_t r, int64_t k, int flip, bool precise)
{
    const int64_t rp = (r + 63) / 64, kp = (k + 63) / 64, x = kp * r * PANEL_BYTES, t = rp * k * PANEL_BYTES, a = rp * r * PANEL_BYTES;
    const int64_t high = flip ? k : r, wide = flip ? r : k;
    const int64_t parts = ((high + NORM_ROWS - 1) / NORM_ROWS) * ((wide + NORM_COLS - 1) / NORM_COLS);
    NsWork w;
    w.x = base, w.xl = w.x + x;
    w.t = w.xl + x, w.t2 = w.t + t;
    w.tl = w.t2 + t, w.tl2 = w.tl + (precise ? t : 0);
    w.e = w.tl2 + (precise ? t : 0), w.g = w.e + a;
    w.el = w.g + a, w.gl = w.el + (precise ? a : 0);
    w.d = (float *)(w.gl + (precise ? a : 0)), w.f = w.d + ((r + 31) & ~31ll);
    w.scale = w.f + ((r + 31) & ~31ll);
    w.squares = (double *)(w.scale + 32);
    w.bytes = (uint8_t *)(w.squares + ((parts + 15) & ~15ll)) - base;
    return w;
}

// The matrix of this workgroup, and which of the matrix's workgroups it is.
__device__ static inline int ns_find(const NsLaunch &l, int id, int *piece)
{
    int i = 0;
    while (i + 1 < l.count && id >= l.m[i + 1].first) i++;
    *piece = id - l.m[i].first;
    return i;
}

__device__ static inline float ns_read(const uint8_t *from, int64_t i, int dtype)
{
    if (dtype == TFTQ_F32) return ((const float *)from)[i];
    if (dtype == TFTQ_F16) return (float)((const _Float16 *)from)[i];
    return (float)((const __bf16 *)from)[i];
}
// The momentum's next value and the update that is orthogonalised.
__device__ static inline float ns_momentum(float m, float g, const NsParams &p) { return m * p.momentum + (1.f - p.momentum) * g; }
__device__ static inline float ns_update(float m, float g, const NsParams &p) { return p.nesterov ? g + p.momentum * (m - g) : m; }

// momentum <- its next value; the sums of the squares of u, one for 64 x 1024 elements, in 64 bits: no
// gradient's norm leaves their range, and the order of the additions is always the same.
__global__ __launch_bounds__(256) void k_ns_squares(const NsLaunch l, const NsParams p, int precise)
{
    __shared__ double sums[4];
    int piece;
    const NsMatrix m = l.m[ns_find(l, blockIdx.x, &piece)];
    const int high = m.flip ? m.cols : m.rows, wide = m.flip ? m.rows : m.cols;
    const int across = (wide + NORM_COLS - 1) / NORM_COLS;
    const int row0 = piece / across * NORM_ROWS, col0 = piece % across * NORM_COLS;
    const int rows = min(NORM_ROWS, high - row0);
    double sum = 0;
    for (int c = threadIdx.x; c < NORM_COLS && col0 + c < wide; c += 256)
#pragma unroll 4
        for (int r = 0; r < rows; r++) {
            float u = ns_read(m.in, (row0 + r) * m.ld_in + col0 + c, p.in_dtype);
            if (m.momentum) {
                float *at = m.momentum + (row0 + r) * m.ld_momentum + col0 + c;
                const float next = ns_momentum(*at, u, p);
                *at = next;
                u = ns_update(next, u, p);
            }
            sum += (double)u * (double)u;
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

// X and X^T in panels from u / |u|, a square of 64 per workgroup.
__global__ __launch_bounds__(256) void k_ns_start(const NsLaunch l, const NsParams p, int precise)
{
    __shared__ float tile[64][65];
    __shared__ double sums[4];
    int piece;
    const NsMatrix m = l.m[ns_find(l, blockIdx.x, &piece)];
    const NsWork w = ns_work(m.work, m.rows, m.cols, m.flip, precise);
    const int across = (m.cols + 63) / 64;
    const int row0 = piece / across * 64, col0 = piece % across * 64;
    const int high = m.flip ? m.cols : m.rows, wide = m.flip ? m.rows : m.cols;
    const int parts = (high + NORM_ROWS - 1) / NORM_ROWS * ((wide + NORM_COLS - 1) / NORM_COLS);
    double sum = 0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += w.squares[i];
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    const double norm = sqrt(sums[0] + sums[1] + sums[2] + sums[3]);
    const double by = 1.0 / (norm <= (double)p.eps ? (double)p.eps : norm);  // a NaN stays one
    const float scale = ns_scale(norm, p);
    if (piece == 0 && threadIdx.x == 0) *w.scale = scale;

    // read along the rows of the matrix as it lies
    const int at_row = m.flip ? col0 : row0, at_col = m.flip ? row0 : col0;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
        const int r = i >> 6, c = i & 63;
        float v = 0.f;
        if (at_row + r < high && at_col + c < wide) {
            float u = ns_read(m.in, (at_row + r) * m.ld_in + at_col + c, p.in_dtype);
            if (m.momentum) u = ns_update(m.momentum[(at_row + r) * m.ld_momentum + at_col + c], u, p);
            v = (float)(u * by);
        }
        if (m.flip) tile[c][r] = v;
        else tile[r][c] = v;
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

// 8 neighbouring results to the list's matrix: the row, the first column and how many of them exist.
__device__ static inline void ns_put(const NsMatrix m, const NsParams p, int64_t row, int64_t col, int n, const float *v)
{
    const int64_t at = row * m.ld_out + col;
    if (p.out_dtype == TFTQ_F32) {
        float *to = (float *)m.out + at;
        const bool vector = m.whole_out && n >= 8;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            tile_f4 o = {0.f, 0.f, 0.f, 0.f};
            if (p.update && vector) o = ((const tile_f4 *)to)[h];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int q = 4 * h + i;
                if (p.update && !vector && q < n) o[i] = to[q];
                o[i] = p.update ? p.keep * o[i] - m.step * v[q] : v[q];
                if (!vector && q < n) to[q] = o[i];
            }
            if (vector) ((tile_f4 *)to)[h] = o;
        }
        return;
    }
    uint16_t *to = (uint16_t *)m.out + at;
    const bool half = p.out_dtype == TFTQ_F16;
    typedef uint16_t s8 __attribute__((ext_vector_type(8)));
    s8 o;
    const bool vector = m.whole_out && n >= 8;
    if (p.update && vector) o = *(const s8 *)to;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float r = v[i];
        if (p.update) {
            if (!vector) o[i] = i < n ? to[i] : (uint16_t)0;
            const float old = half ? (float)__builtin_bit_cast(_Float16, (uint16_t)o[i]) : (float)__builtin_bit_cast(__bf16, (uint16_t)o[i]);
            r = p.keep * old - m.step * r;
        }
        o[i] = half ? __builtin_bit_cast(uint16_t, (_Float16)r) : __builtin_bit_cast(uint16_t, (__bf16)r);
        if (!vector && i < n) to[i] = o[i];
    }
    if (vector) *(s8 *)to = o;
}

enum { NS_A, NS_B, NS_X };

template <class T, int WHAT, bool PRECISE>
__global__ __launch_bounds__(T::THREADS) void k_ns_product(const NsLaunch l, const NsParams p, int turn)
{
    __shared__ __attribute__((aligned(128))) uint8_t lds[T::LDS];
    int piece;
    const NsMatrix m = l.m[ns_find(l, tile_piece(blockIdx.x, gridDim.x), &piece)];
    const int r = m.rows, k = m.cols, rp = (r + 63) >> 6;
    const NsWork w = ns_work(m.work, r, k, m.flip, PRECISE);
    int tm, tn;
    if (WHAT == NS_X) {
        tile_place(piece, (r + T::ROWS - 1) / T::ROWS, (k + T::COLS - 1) / T::COLS, &tm, &tn);
    } else {  // column tn of the upper triangle has tn + 1 tiles
        tn = (int)((sqrtf(8.f * piece + 1.f) - 1.f) * 0.5f);
        while ((tn + 1) * (tn + 2) / 2 <= piece) tn++;
        while (tn * (tn + 1) / 2 > piece) tn--;
        tm = piece - tn * (tn + 1) / 2;
    }
    const int row0 = tm * T::ROWS, col0 = tn * T::COLS;

    const uint8_t *ah = WHAT == NS_A ? w.x : WHAT == NS_B ? w.e : w.g, *al = WHAT == NS_A ? w.xl : WHAT == NS_B ? w.el : w.gl;
    const uint8_t *bh = WHAT == NS_A ? w.x : WHAT == NS_B ? w.e : turn ? w.t2 : w.t, *bl = WHAT == NS_A ? w.xl : WHAT == NS_B ? w.el : turn ? w.tl2 : w.tl;
    const int panels = WHAT == NS_A ? (k + 63) >> 6 : rp, b_rows = WHAT == NS_X ? k : r;
    T t;
    auto place = [&](int, int *r0, int *c0) { *r0 = row0, *c0 = col0; };
    auto done = [](int, int) {};
    if constexpr (PRECISE) t.multiply(TileTriple{{ah, al, bh, bl, r, b_rows, panels}}, 3 * panels, 1, place, lds, done);
    else t.multiply(TilePair{{ah, nullptr, r}, {bh, nullptr, b_rows}}, panels, 1, place, lds, done);

    // The result's panels: along its rows, and along its columns (its transpose), each with its remainder.
    uint8_t *out = WHAT == NS_A ? w.e : WHAT == NS_B ? w.g : w.x, *out_l = WHAT == NS_A ? w.el : WHAT == NS_B ? w.gl : w.xl;
    uint8_t *flip = WHAT != NS_X ? out : turn ? w.t : w.t2, *flip_l = WHAT != NS_X ? out_l : turn ? w.tl : w.tl2;
    const float scale_x = *w.scale, per_x = 1.f / scale_x;  // powers of two
    const float scale = WHAT == NS_A ? SCALE_E : WHAT == NS_B ? SCALE_G : scale_x;
    constexpr bool LOW = PRECISE || WHAT == NS_X;
    const int cols = WHAT == NS_X ? k : r, padded = (cols + 63) & ~63;
    const bool last = WHAT == NS_X && p.last, mirror = WHAT == NS_X ? !last || m.flip : tm != tn;
    const int lane = threadIdx.x & 63;

    t.store_strips(row0, col0, lds, [&](float *strip, int row, int col) {
        constexpr int ACROSS = T::WN / 8;
        const int c = lane % ACROSS * 8, j0 = col + c;
#pragma unroll 1
        for (int q = lane / ACROSS; q < 32; q += 64 / ACROSS) {
            const int i = row + q;
            float *v = strip + q * T::PITCH + c;
            const bool inside = i < r && j0 < padded;
            const int64_t at = ((int64_t)(j0 >> 6) * r + i) * PANEL_BYTES + (j0 & 63) * 2;
            float o[8];
            if (WHAT == NS_A) {
#pragma unroll
                for (int n = 0; n < 8; n++) {
                    o[n] = v[n] * per_x * per_x;
                    if (i == j0 + n && i < r) w.d[i] = o[n];
                }
            } else if (inside) {
                ns_h8 hi = *(const ns_h8 *)((WHAT == NS_B ? w.e : w.x) + at), lo = hi;
                if (LOW) lo = *(const ns_h8 *)((WHAT == NS_B ? w.el : w.xl) + at);
                const float di = WHAT == NS_B ? w.d[i] : p.a + w.f[i];
#pragma unroll
                for (int n = 0; n < 8; n++) {
                    const float old = ((float)hi[n] + (LOW ? (float)lo[n] : 0.f)) * (WHAT == NS_B ? 1.f / SCALE_E : per_x);
                    if (WHAT == NS_B) {
                        const float dj = j0 + n < r ? w.d[j0 + n] : 0.f, square = v[n] * (1.f / (SCALE_E * SCALE_E));
                        if (i == j0 + n) w.f[i] = p.b * di + p.c * (square + di * di);
                        o[n] = p.b * old + p.c * (square + (di + dj) * old);
                    } else {
                        o[n] = di * old + v[n] * (1.f / SCALE_G) * per_x;
                    }
                }
            }
            ns_h8 hi, lo;
#pragma unroll
            for (int n = 0; n < 8; n++) {
                if (!inside || j0 + n >= cols || (WHAT != NS_X && i == j0 + n)) o[n] = 0.f;
                _Float16 a, b;
                ns_split(o[n], scale, &a, &b);
                hi[n] = a, lo[n] = b;
                v[n] = o[n];
            }
            if (last) {
                if (!m.flip && inside) ns_put(m, p, i, j0, cols - j0, o);
            } else if (inside) {
                *(ns_h8 *)(out + at) = hi;
                if (LOW) *(ns_h8 *)(out_l + at) = lo;
            }
        }
        T::wave_fence();
        if (!mirror) return;
        // the same values down the columns, 8 rows of a column per lane
#pragma unroll 1
        for (int q = lane; q < T::WN * 4; q += 64) {
            const int i0 = row + (q & 3) * 8, j = col + (q >> 2);
            if (j >= cols || i0 >= rp * 64) continue;
            float o[8];
            ns_h8 hi, lo;
#pragma unroll
            for (int n = 0; n < 8; n++) {
                o[n] = strip[((q & 3) * 8 + n) * T::PITCH + (q >> 2)];
                _Float16 a, b;
                ns_split(o[n], scale, &a, &b);
                hi[n] = a, lo[n] = b;
            }
            if (last) {
                if (i0 < r) ns_put(m, p, j, i0, r - i0, o);
                continue;
            }
            const int64_t at = ((int64_t)(i0 >> 6) * cols + j) * PANEL_BYTES + (i0 & 63) * 2;
            *(ns_h8 *)(flip + at) = hi;
            if (PRECISE) *(ns_h8 *)(flip_l + at) = lo;
        }
    });
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <class F>
static int launch_over(NsLaunch &l, F workgroups, const void *kernel, int threads, const NsParams &p, int extra, hipStream_t st)
{
    int64_t total = 0;
    for (int i = 0; i < l.count; i++) {
        l.m[i].first = (int)total;
        total += workgroups(l.m[i]);
        if (total > (1 << 22)) return TFTQ_E_SHAPE;
    }
    void *args[] = {(void *)&l, (void *)&p, (void *)&extra};
    return (int)hipLaunchKernel(kernel, dim3((unsigned)total), dim3(threads), args, 0, st);
}

static int64_t tiles(const NsMatrix &m, int what, int size)
{
    const int64_t r = (m.rows + size - 1) / size, k = (m.cols + size - 1) / size;
    return what == NS_X ? r * k : r * (r + 1) / 2;
}

template <class T, int WHAT>
static int launch_product(NsLaunch &l, bool precise, const NsParams &p, int turn, hipStream_t st)
{
    const void *k = precise ? (const void *)k_ns_product<T, WHAT, true> : (const void *)k_ns_product<T, WHAT, false>;
    return launch_over(l, [](const NsMatrix &m) { return tiles(m, WHAT, T::ROWS); }, k, T::THREADS, p, turn, st);
}

// One of the three products for all matrices of a launch, with the largest tiles that give most compute units one.
template <int WHAT>
static int product(NsLaunch &l, bool precise, const NsParams &p, int turn, hipStream_t st)
{
    int64_t big = 0, middle = 0;
    for (int i = 0; i < l.count; i++) big += tiles(l.m[i], WHAT, 256), middle += tiles(l.m[i], WHAT, 128);
    if (big >= 160) return launch_product<Tile<256, 256, 2, 4, false>, WHAT>(l, precise, p, turn, st);
    if (middle >= 160) return launch_product<Tile<128, 128, 2, 2, false>, WHAT>(l, precise, p, turn, st);
    return launch_product<Tile<64, 64, 2, 2, false>, WHAT>(l, precise, p, turn, st);
}

static bool ns_shapes_ok(int n, const int64_t *shapes)
{
    for (int i = 0; i < 2 * n; i++)
        if (shapes[i] < 0 || shapes[i] > NS_LONGEST) return false;
    return true;
}

// Whether a matrix of r rows (columns, if these are fewer) takes three products.  The errors of the one of 11
// bits are those of many roundings, and average: 2e-3 at most in 20 draws of each spectrum from 32 rows
// on, but 8e-3 for a 3x5 matrix with singular values of 1 and 0.02.  A matrix of fewer than 64 rows is
// one tile high, and its products wait for memory, not for the matrix cores.
static bool ns_precise(int64_t r, int precise) { return precise || r < 64; }

// f(the matrices of one launch, how many, whether they take three products, bytes of workspace) for the whole list.
template <class F>
static int ns_parts(int n, const int64_t *shapes, int precise, F f)
{
    for (int kind = 0; kind < 2; kind++) {
        int at[NS_MOST], count = 0;
        int64_t bytes = 0;
        for (int i = 0; i < n; i++) {
            const int64_t a = shapes[2 * i], b = shapes[2 * i + 1], r = a < b ? a : b;
            if (r == 0 || ns_precise(r, precise) != (kind != 0)) continue;
            bytes += ns_work(nullptr, r, a < b ? b : a, a > b, kind != 0).bytes;
            at[count++] = i;
            if (count < NS_MOST) continue;
            if (const int rc = f(at, count, kind != 0, bytes)) return rc;
            count = 0, bytes = 0;
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
    ns_parts(n, shapes, precise, [&](const int *, int, bool, int64_t bytes) {
        most = std::max(most, bytes);
        return 0;
    });
    return most;
}

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
    if (needed == 0) return 0;
    if (workspace_bytes < needed) return TFTQ_E_SIZE;
    if (!workspace || ((uintptr_t)workspace & 127)) return TFTQ_E_ARG;
    DeviceScope scope(device);
    if (scope.err != hipSuccess) return (int)scope.err;
    hipStream_t st = (hipStream_t)stream;
    const int out_size = s.out_dtype == TFTQ_F32 ? 4 : 2;

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
            m.whole_out = m.ld_out * out_size % 16 == 0 && (uintptr_t)m.out % 16 == 0;
            m.step = s.steps ? s.steps[i] : 0.f;
            m.work = work;
            work += ns_work(nullptr, m.rows, m.cols, m.flip, precise).bytes;
        }
        float growth = 1.f;
        for (int it = 0; it < s.iterations; it++) growth *= fmaxf(1.f, fabsf(s.coefficients[3 * it]));
        NsParams p = {s.momentum, s.keep, 0, 0, 0, s.eps, growth, s.nesterov, s.in_dtype, s.out_dtype, s.steps != nullptr, 0};
        int rc = launch_over(l, [](const NsMatrix &m) {
            const int64_t high = m.flip ? m.cols : m.rows, wide = m.flip ? m.rows : m.cols;
            return (high + NORM_ROWS - 1) / NORM_ROWS * ((wide + NORM_COLS - 1) / NORM_COLS);
        }, (const void *)k_ns_squares, 256, p, precise, st);
        if (rc) return rc;
        rc = launch_over(l, [](const NsMatrix &m) { return (int64_t)((m.rows + 63) / 64) * ((m.cols + 63) / 64); },
                         (const void *)k_ns_start, 256, p, precise, st);
        if (rc) return rc;
        for (int it = 0; it < s.iterations; it++) {
            p.a = s.coefficients[3 * it], p.b = s.coefficients[3 * it + 1], p.c = s.coefficients[3 * it + 2];
            p.last = it + 1 == s.iterations;
            if ((rc = product<NS_A>(l, precise, p, it & 1, st)) || (rc = product<NS_B>(l, precise, p, it & 1, st)) ||
                (rc = product<NS_X>(l, precise, p, it & 1, st)))
                return rc;
        }
        return 0;
    });
}
