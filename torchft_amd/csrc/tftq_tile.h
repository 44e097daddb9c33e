// A tile of a product of two matrices whose rows are contracted, C[i][j] = sum_k A[i][k] B[j][k],
// on the matrix cores of gfx950.  Shared by the product of 4-bit microscaled matrices
// (tftq_mxfp4_product.hip) and the products of the Newton-Schulz iteration (tftq_orthogonal.hip).
//
// Both operands lie in panels: panel s of a matrix of R rows is R pieces of 128 bytes, one after the
// other, that hold columns [s W, (s + 1) W) of every row (W = 64 for fp16, 256 for 4-bit codes), and is
// zero past the last column.  128 bytes of a row are what a workgroup multiplies between two barriers,
// so a tile's rows of a panel are one run of memory, whatever the matrix's width.
//
// The two types need the same bytes in the same lanes: v_mfma_f32_32x32x16_f16 takes 8 elements and
// v_mfma_scale_f32_32x32x64_f8f6f4 takes 32 codes, 16 bytes either way, of row lane % 32 from half
// lane / 32 of a slice of 32 bytes.  One kernel body therefore serves both; the 4-bit one also hands the
// instruction the scale of the lane's 32 codes.
//
// Staging: loads straight into LDS, 16 bytes per lane and 8 rows per instruction, one barrier per panel and
// two buffers (small tiles: three); a buffer's next panel is loaded from the moment when everybody has read
// the one that it holds.  A wavefront's bytes land in LDS in lane order, so the order in which lanes take
// the 16-byte pieces of their row is what arranges the buffer: piece p of row r lies at place p ^ (r % 8), and the 8 lanes that one cycle of ds_read_b128
// serves, 8 neighbouring rows, find their pieces in 8 different groups of banks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <utility>

typedef int tile_i4 __attribute__((ext_vector_type(4)));
typedef uint32_t tile_u2 __attribute__((ext_vector_type(2)));
typedef int tile_i8 __attribute__((ext_vector_type(8)));
typedef float tile_f4 __attribute__((ext_vector_type(4)));
typedef float tile_f16 __attribute__((ext_vector_type(16)));
typedef _Float16 tile_h8 __attribute__((ext_vector_type(8)));

constexpr int PANEL_BYTES = 128;

// One operand: its panels and, for 4-bit codes, the scales that go with them: 8 bytes for every row of
// a panel, panel by panel, with an even number of rows in each.
struct TileOperand {
    const uint8_t *panels;
    const uint8_t *scales;
    int rows;
};

// Two operands as fp16 numbers and what their rounding left, as fp16 numbers too: the products high x
// high, low x high and high x low, one after the other, as one sum over three times the panels.
struct TileSplit {
    const uint8_t *a_high, *a_low, *b_high, *b_low;
    int a_rows, b_rows, panels;
};
// What a step of a tile's loop multiplies: panel s of either operand.
struct TilePanels {
    const uint8_t *a, *b, *a_scales, *b_scales;
};
struct TilePair {  // one product
    TileOperand a, b;
    __device__ int a_rows() const { return a.rows; }
    __device__ int b_rows() const { return b.rows; }
    __device__ TilePanels at(int s) const
    {
        return {a.panels + (int64_t)s * a.rows * PANEL_BYTES, b.panels + (int64_t)s * b.rows * PANEL_BYTES,
                a.scales + (int64_t)s * ((a.rows + 1) & ~1) * 8, b.scales + (int64_t)s * ((b.rows + 1) & ~1) * 8};
    }
};
struct TileTriple {  // three
    TileSplit o;
    __device__ int a_rows() const { return o.a_rows; }
    __device__ int b_rows() const { return o.b_rows; }
    __device__ TilePanels at(int s) const
    {
        const uint8_t *a = o.a_high, *b = o.b_high;
        if (s >= 2 * o.panels) b = o.b_low, s -= 2 * o.panels;
        else if (s >= o.panels) a = o.a_low, s -= o.panels;
        return {a + (int64_t)s * o.a_rows * PANEL_BYTES, b + (int64_t)s * o.b_rows * PANEL_BYTES, nullptr, nullptr};
    }
};

// A buffer of `bytes` bytes (what lies past them reads as zero), and a load of 16 bytes per lane from it
// into LDS, in lane order from `lds` on.  `more`, in a scalar register, counts in the check of the end as `at` does
// (1024 bytes, at < 1024: all zeros from more = 1024 on, and half of the lanes at 512), also where it alone
// passes the end.  (The global instruction that does the same makes the compiler wait for every LDS read in flight at the
// next use of one.)
__device__ static inline __amdgpu_buffer_rsrc_t tile_buffer(const uint8_t *from, int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)from, 0, bytes, 0x00020000);
}
__device__ static inline void tile_load16(__amdgpu_buffer_rsrc_t from, int at, int more, uint8_t *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)lds, 16, at, more, 0, 0);
}

// f(0), f(1) and so on, constants: arrays that f indexes with them stay in registers, whatever f's size
// (loops of large bodies are unrolled too late for that).
template <class F, int... I>
__device__ static __forceinline__ void tile_each(std::integer_sequence<int, I...>, F f)
{
    (f(std::integral_constant<int, I>()), ...);
}

// The wavefront's number in its workgroup, in a scalar register.
__device__ static inline int tile_wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// BM x BN values of C by WGM x WGN wavefronts, each of them TM x TN squares of 32.  BUFFERS: panels in LDS;
// with more than two a panel is loaded BUFFERS - 1 panels ahead, for small tiles, which multiply a panel in
// less time than it takes to come (tiles of 64 x 64 with 2, 3 and 4: 1024x1024 orthogonalised 382, 292,
// 293 us; 4-bit 128x4096x14336 33.5, 28.1, 28.1; 4 leave LDS for fewer tiles to a unit).
template <int BM, int BN, int WGM, int WGN, bool FP4, int BUFFERS = 2>
struct Tile {
    static constexpr int ROWS = BM, COLS = BN, WAVES = WGM * WGN, THREADS = 64 * WAVES;
    static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
    // the first half of the wavefronts loads a's scales of a panel, the other half b's, 1024 bytes each
    // (zeros past the last ones: without a branch in the loop)
    static constexpr int SCALES = WAVES / 2 * 1024;
    static constexpr int BUFFER = (BM + BN) * PANEL_BYTES + (FP4 ? 2 * SCALES : 0);
    // a wavefront's strip of 32 rows of results, behind the buffers' use (store_strips)
    static constexpr int PITCH = WN + 4;
    static constexpr int LDS = BUFFERS * BUFFER > WAVES * 32 * PITCH * 4 ? BUFFERS * BUFFER : WAVES * 32 * PITCH * 4;
    static constexpr int LDS_PIECES = BUFFERS * BUFFER + WAVES * 2048, PIECES_AT = BUFFERS * BUFFER;
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "every wavefront loads the same number of rows");
    static_assert(LDS <= 160 * 1024 && LDS_PIECES <= 160 * 1024 && BM * 8 <= SCALES && BN * 8 <= SCALES, "");

    tile_f16 acc[TM][TN];

    __device__ void zero()
    {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
    }

    // What a step of the loop loads: a panel of the rows of a tile.  Rows past the last one read as zero.
    struct Step {
        const uint8_t *a, *b, *scales;
        int a_bytes, b_bytes, scale_bytes;
    };
    template <class P>
    __device__ static Step step(const P &p, int s, int row0, int col0)
    {
        const TilePanels at = p.at(s);
        const int rows = min(p.a_rows() - row0, BM), cols = min(p.b_rows() - col0, BN);
        Step t = {at.a + (int64_t)row0 * PANEL_BYTES, at.b + (int64_t)col0 * PANEL_BYTES, nullptr, rows * PANEL_BYTES, cols * PANEL_BYTES, 0};
        if (FP4) {  // two rows per lane: a's for the first half of the wavefronts, b's for the other
            const bool m = tile_wave() < WAVES / 2;
            t.scales = m ? at.a_scales + (int64_t)row0 * 8 : at.b_scales + (int64_t)col0 * 8;
            t.scale_bytes = (((m ? rows : cols) + 1) & ~1) * 8;
        }
        return t;
    }
    // Part `part` of `parts` of a wavefront's loads of a step, 8 rows an instruction.
    static constexpr int LOADS_M = BM / (8 * WAVES), LOADS_N = BN / (8 * WAVES), LOADS = LOADS_M + LOADS_N + (FP4 ? 1 : 0);
    __device__ static void load_part(const Step &t, int at, uint8_t *buf, int part, int parts)
    {
        const int wave = tile_wave();
        const __amdgpu_buffer_rsrc_t a = tile_buffer(t.a, t.a_bytes), b = tile_buffer(t.b, t.b_bytes);
#pragma unroll
        for (int n = 0; n < LOADS_M + LOADS_N; n++) {
            if (n * parts / (LOADS_M + LOADS_N) != part) continue;
            constexpr int EACH = WAVES * 8 * PANEL_BYTES;
            if (n < LOADS_M) tile_load16(a, at, n * EACH, buf + n * EACH + wave * 8 * PANEL_BYTES);
            else tile_load16(b, at, (n - LOADS_M) * EACH, buf + (BM * PANEL_BYTES + (n - LOADS_M) * EACH) + wave * 8 * PANEL_BYTES);
        }
        if (FP4 && part == 0)
            tile_load16(tile_buffer(t.scales, t.scale_bytes), (threadIdx.x & 63) * 16, wave % (WAVES / 2) * 1024,
                        buf + (BM + BN) * PANEL_BYTES + wave * 1024);
    }

    // The 16 bytes of every row and column that slice q of a panel takes, and the scales of a panel.
    struct Slice {
        tile_i4 a[TM], b[TN];
    };
    struct Scales {
        uint32_t a[TM][2], b[TN][2];
    };

    // The products over `panels` panels of `tiles` tiles, one after the other: place(t, &row0, &col0) says
    // where tile t lies, done(row0, col0) takes its values out of acc.  Every wavefront of the workgroup
    // calls it with the same arguments.
    //
    // Slice q + 1 is read from LDS while slice q is multiplied, and the first slice of the next panel while
    // the last one of this panel is: the barrier between the panels stands before that last slice, whose
    // operands are in registers by then, so the matrix cores have work on both sides of it, and the
    // loads of the panel after the next, half of them behind it and half in the next slice, have the time
    // to the next barrier.  The order (a few reads, a few loads, TN products, TM times a slice) is written
    // out and kept.  A tile's first panels are on their way while the last tile's values are stored.
    template <class P, class G, class D>
    __device__ __forceinline__ void multiply(const P &p, int panels, int tiles, G place, uint8_t *lds, D done)
    {
        const int lane = threadIdx.x & 63, wave = tile_wave();
        const int wm = wave / WGN * WM, wn = wave % WGN * WN;
        const int in_row = lane & 31, half = lane >> 5;
        int at[4];
#pragma unroll
        for (int q = 0; q < 4; q++) at[q] = ((2 * q + half) ^ (lane & 7)) * 16;
        const int a_at = (wm + in_row) * PANEL_BYTES, b_at = (BM + wn + in_row) * PANEL_BYTES;
        const int load_at = (wave * 8 + (lane >> 3)) * PANEL_BYTES + ((lane & 7) ^ (lane >> 3)) * 16;
        Slice slice[2];
        Scales scale[2];

        // the tile that is multiplied; the panel after the next one of its, or of a later tile's
        int tile = 0, row0, col0, ahead = 0, ahead_panel = 0, ahead_row, ahead_col;
        place(0, &row0, &col0);
        ahead_row = row0, ahead_col = col0;
        auto advance = [&] {
            if (++ahead_panel < panels) return;
            if (ahead + 1 < tiles) place(++ahead, &ahead_row, &ahead_col), ahead_panel = 0;
            else ahead_panel = panels - 1;  // the last panel is loaded again: no branch among the products
        };
        zero();
        if (panels <= 0) {
            for (; tile < tiles; tile++) {
                place(tile, &row0, &col0);
                done(row0, col0);
            }
            return;
        }
        load_part(step(p, 0, row0, col0), load_at, lds, 0, 1);
        Step next;
        if constexpr (BUFFERS == 2) {
            advance();
            next = step(p, ahead_panel, ahead_row, ahead_col);
            landed<0>();
#pragma unroll
            for (int i = 0; i < TM; i++) load_part(next, load_at, lds + BUFFER, i, 2 * TM);
        } else {
#pragma unroll
            for (int n = 1; n < BUFFERS; n++) {
                advance();
                load_part(step(p, ahead_panel, ahead_row, ahead_col), load_at, lds + n * BUFFER, 0, 1);
            }
            landed<(BUFFERS - 1) * LOADS>();
        }
        advance();
        Step later = step(p, ahead_panel, ahead_row, ahead_col);
        int cur = 0, then = BUFFER;
#pragma unroll
        for (int i = 0; i < TM; i++) read_part(slice[0], lds, a_at + at[0], b_at + at[0], i);
        if (FP4) read_scales(scale[0], lds, wm + in_row, wn + in_row, half);
        for (int s = 0;;) {
            const uint8_t *buf = lds + cur;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (q == 3) {
                    // the next panel has landed, and everybody has read all of this one
                    landed<(BUFFERS - 2) * LOADS>();
                    buf = lds + then;
                    if (FP4) read_scales(scale[1], buf, wm + in_row, wn + in_row, half);
                }
#pragma unroll
                for (int i = 0; i < TM; i++) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int to = (q + 1) & 3;
                    read_part(slice[(q + 1) & 1], buf, a_at + at[to], b_at + at[to], i);
                    if (BUFFERS == 2 && q == 0) load_part(next, load_at, lds + then, TM + i, 2 * TM);
                    if (q == 3) load_part(later, load_at, lds + cur, i, BUFFERS == 2 ? 2 * TM : TM);
#pragma unroll
                    for (int j = 0; j < TN; j++)
                        acc[i][j] = one(slice[q & 1].b[j], slice[q & 1].a[i], acc[i][j], q, scale[0].b[j], scale[0].a[i]);
                }
            }
            if (FP4) scale[0] = scale[1];
            cur = then;
            then = then + BUFFER == BUFFERS * BUFFER ? 0 : then + BUFFER;
            if (++s == panels) {
                done(row0, col0);
                if (++tile == tiles) break;
                place(tile, &row0, &col0);
                zero();
                s = 0;
            }
            if (BUFFERS == 2) next = later;
            advance();
            later = step(p, ahead_panel, ahead_row, ahead_col);
        }
        landed<0>();  // nothing is on its way to LDS any more
    }

    // Waits until all but this wavefront's last N memory operations are done, then for the other wavefronts.
    // Operations are done in the order in which they were issued, and a wavefront issues LOADS of them for
    // every panel, none of them on a condition: with the loads of k later panels issued, a panel has landed
    // when all but k LOADS are done (a tile's stores between them only make the wait longer).
    template <int N>
    __device__ static void landed()
    {
        static_assert(N < 64, "");
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
    }

    // Part `part` of the TM parts of a slice's reads.
    __device__ static void read_part(Slice &f, const uint8_t *buf, int a, int b, int part)
    {
        constexpr int EACH = (TM + TN + TM - 1) / TM;
#pragma unroll
        for (int n = 0; n < EACH; n++) {
            const int at = part * EACH + n;
            if (at < TN) f.b[at] = *(const tile_i4 *)(buf + b + 32 * at * PANEL_BYTES);
            else if (at < TM + TN) f.a[at - TN] = *(const tile_i4 *)(buf + a + 32 * (at - TN) * PANEL_BYTES);
        }
    }
    // Of the 8 scales of a row in a panel the lane needs its half's: bytes 0 and 2 of both words.
    __device__ static void read_scales(Scales &f, const uint8_t *buf, int a, int b, int half)
    {
        const uint8_t *sc = buf + (BM + BN) * PANEL_BYTES;
#pragma unroll
        for (int i = 0; i < TM + TN; i++) {
            const uint64_t v = *(const uint64_t *)(sc + (i < TM ? (a + 32 * i) * 8 : SCALES + (b + 32 * (i - TM)) * 8)) >> (8 * half);
            uint32_t *to = i < TM ? f.a[i] : f.b[i - TM];
            to[0] = (uint32_t)v, to[1] = (uint32_t)(v >> 32);
        }
    }

    __device__ static tile_f16 one(tile_i4 x, tile_i4 y, tile_f16 c, int q, const uint32_t *sx, const uint32_t *sy)
    {
        if constexpr (FP4) {
            const tile_i8 X = {x[0], x[1], x[2], x[3], 0, 0, 0, 0}, Y = {y[0], y[1], y[2], y[3], 0, 0, 0, 0};
            // format 4 is e2m1; slice q's scale is byte 0 (even q) or 2 of word q / 2
            if (q & 1) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(X, Y, c, 4, 4, 2, sx[q >> 1], 2, sy[q >> 1]);
            return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(X, Y, c, 4, 4, 0, sx[q >> 1], 0, sy[q >> 1]);
        } else {
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(tile_h8, x), __builtin_bit_cast(tile_h8, y), c, 0, 0, 0);
        }
    }

    // f(i, strip, row, col) for every 32 x WN values of the wavefront, strip[r * PITCH + c] in LDS being
    // C[row + r][col + c]; before(i, row, col) is called a strip ahead, to load what f needs (i: a constant,
    // so that what they keep from strip to strip stays in registers).  A lane's accumulators hold 4
    // neighbouring values of one row, 8 columns apart (b is the instruction's first operand); from the strip
    // it takes what makes whole 16 bytes of the result.
    template <class B, class F>
    __device__ __forceinline__ void store_strips(int row0, int col0, uint8_t *lds, B before, F f)
    {
        const int wave = tile_wave();
        const int row = row0 + wave / WGN * WM, col = col0 + wave % WGN * WN;
        float *strip = (float *)lds + wave * 32 * PITCH;
        const int lane = threadIdx.x & 63;
        before(std::integral_constant<int, 0>(), row, col);
        tile_each(std::make_integer_sequence<int, TM>(), [&](auto i) __attribute__((always_inline)) {
            if constexpr (i + 1 < TM) before(std::integral_constant<int, i + 1>(), row + 32 * (i + 1), col);
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *(tile_f4 *)(strip + (lane & 31) * PITCH + 32 * j + 8 * g + 4 * (lane >> 5)) =
                        tile_f4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            wave_fence();
            f(i, strip, row + 32 * i, col);
            wave_fence();
        });
    }
    // f(the lane's 16 bytes, row, column) of the results, as elements of SIZE bytes; `to` makes a word of two
    // sums of those of 2.  By way of 2048 bytes of LDS per wavefront beside the buffers: 64 bytes of 32
    // rows at a time, so that 4 lanes have a whole line's half.
    template <int SIZE, class C, class F>
    __device__ __forceinline__ void store_pieces(int row0, int col0, uint8_t *lds, C to, F f)
    {
        constexpr int COLS = 64 / SIZE;
        const int lane = threadIdx.x & 63, wave = tile_wave();
        const int wm = wave / WGN * WM, wn = wave % WGN * WN;
        uint8_t *own = lds + wave * 2048;
        const int row = lane & 31, half = lane >> 5;
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int c = 0; c < WN / COLS; c++) {
                // 16 bytes of a row lie at place (their number) ^ (row / 4 % 4)
#pragma unroll
                for (int g = 0; g < COLS / 8; g++) {
                    const int first = c * COLS + 8 * g;
                    const tile_f16 &from = acc[i][first / 32];
                    const int r = first % 32 / 8 * 4;
                    if constexpr (SIZE == 2) {
                        const tile_u2 v = {to(from[r], from[r + 1]), to(from[r + 2], from[r + 3])};
                        *(tile_u2 *)(own + row * 64 + ((g ^ (row >> 2)) & 3) * 16 + half * 8) = v;
                    } else {
                        *(tile_f4 *)(own + row * 64 + (((2 * g + half) ^ (row >> 2)) & 3) * 16) = tile_f4{from[r], from[r + 1], from[r + 2], from[r + 3]};
                    }
                }
                wave_fence();
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int at = n * 16 + (lane >> 2);
                    const tile_i4 v = *(const tile_i4 *)(own + at * 64 + (((lane & 3) ^ (at >> 2)) & 3) * 16);
                    f(v, row0 + wm + 32 * i + at, col0 + wn + c * COLS + (lane & 3) * (16 / SIZE));
                }
                wave_fence();
            }
    }

    // LDS of a wavefront's own: its accesses are performed in order, the compiler keeps them so.
    __device__ static void wave_fence()
    {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
};

// Workgroup `id` of `count` -> its piece of the work: ids go to the 8 XCDs in turn, and each XCD gets
// one run of neighbouring pieces (an operand's rows are then in one L2, not in eight).
__device__ static inline int tile_piece(int id, int count)
{
    const int xcd = id & 7, n = id >> 3, whole = count >> 3, more = count & 7;
    return xcd * whole + min(xcd, more) + n;
}
// The same for `groups` workgroups that share `count` pieces (no fewer than workgroups): the first of the
// workgroup's pieces, how far the next one is, and how many it has.
__device__ static inline int tile_pieces(int id, int groups, int count, int *apart, int *pieces)
{
    const int xcd = id & 7, n = id >> 3, whole = count >> 3, more = count & 7;
    *apart = (groups - xcd + 7) >> 3;
    *pieces = (whole + (xcd < more) - n + *apart - 1) / *apart;
    return xcd * whole + min(xcd, more) + n;
}

// Piece -> (row tile, column tile): bands of 8 row tiles, column by column inside a band, so that
// the ~32 tiles that run on an XCD at once share 8 row tiles and 4 column tiles.
__device__ static inline void tile_place(int piece, int tiles_m, int tiles_n, int *tm, int *tn)
{
    const int band = piece / (8 * tiles_n), first = band * 8, height = min(8, tiles_m - first);
    const int in = piece - band * 8 * tiles_n;
    *tn = in / height;
    *tm = first + in % height;
}

// A size of tiles.  `at_once`: the tiles that a compute unit runs at once; `cost`: what a panel of them all
// takes then, `one` with one tile to a unit, a panel of one tile of 256 x 256 on every unit being 1.  From
// launches that fill all units (8192^3, fp16, TFLOP/s: 256x256 1230, 192x256 1190, 192x192 1040, 128x128
// 1000, 64x64 760; 4-bit, 256x256 4600, 192x256 4100, 128x128 3580, 64x64 1870) and from short ones (4-bit, us, tiles
// of 256, 128, 64: 256x4096x4096 22.8, 12.4, 9.6; 256x14336x4096 24.8, 16.5, 22.5; 2048x5632x2048 18.7, 21.0, 31.4).
// 128x128 is 0.61 by its rate, but 3 to a unit take 1.02 (a list of products of depth 2048 in 696 tiles
// 79 us, in 216 of 256x256 71), and 192x256 0.775, but with a round more than 256x256 it loses (4-bit
// 14336x4096x8192 230 us, 221; X of 4096x14336 572, 552; with fewer, 4-bit 6144x6144x6144, 112, 122).
struct TileShape {
    int high, wide, at_once;
    double one, cost;
};
constexpr TileShape TILES_256 = {256, 256, 1, 1.0, 1.0}, TILES_192X256 = {192, 256, 1, 0.82, 0.82},
                    TILES_192 = {192, 192, 1, 0.665, 0.665}, TILES_128 = {128, 128, 2, 0.41, 0.68},
                    TILES_64 = {64, 64, 3, 0.22, 0.30}, TILES_64_FP4 = {64, 64, 2, 0.26, 0.31};

// About how many panels of a 256 x 256 tile `count` tiles of that size take together: `work` panels in
// all, `longest` the longest of them.  Storing a tile's values and waiting for its first operands takes
// about as long as 4 panels.
static inline double tile_time(const TileShape &t, double count, double work, double longest)
{
    const int64_t units = ((int64_t)count + 255) / 256;
    const double each = work / count + 4;
    const double alone = units < t.at_once ? t.one + (t.cost - t.one) * (units - 1) / (t.at_once - 1) : t.cost;
    const double rounds = units < t.at_once ? 1 : (double)units / t.at_once;
    return std::max(rounds * each, longest + 4) * alone;
}
