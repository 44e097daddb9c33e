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
// Staging: global_load_lds of 16 bytes per lane, 8 rows per instruction, two buffers, one barrier per
// panel; the loads of panel s + 1 run while panel s is multiplied.  A wavefront's bytes land in LDS in
// lane order, so the order in which lanes take the 16-byte pieces of their row is what arranges the
// buffer: piece p of row r lies at place p ^ (r % 8), and the 8 lanes that one cycle of ds_read_b128
// serves, 8 neighbouring rows, find their pieces in 8 different groups of banks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef int tile_i4 __attribute__((ext_vector_type(4)));
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

__device__ static inline void tile_load16(const uint8_t *from, uint8_t *lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// The wavefront's number in its workgroup, in a scalar register.
__device__ static inline int tile_wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// BM x BN values of C by WGM x WGN wavefronts, each of them TM x TN squares of 32.
template <int BM, int BN, int WGM, int WGN, bool FP4>
struct Tile {
    static constexpr int ROWS = BM, COLS = BN, WAVES = WGM * WGN, THREADS = 64 * WAVES;
    static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / 32, TN = WN / 32;
    static constexpr int SCALES_M = BM * 8 < 1024 ? 1024 : BM * 8, SCALES_N = BN * 8 < 1024 ? 1024 : BN * 8;
    static constexpr int BUFFER = (BM + BN) * PANEL_BYTES + (FP4 ? SCALES_M + SCALES_N : 0);
    // a wavefront's strip of 32 rows of results, behind the buffers' use (store_strips)
    static constexpr int PITCH = WN + 4;
    static constexpr int LDS = 2 * BUFFER > WAVES * 32 * PITCH * 4 ? 2 * BUFFER : WAVES * 32 * PITCH * 4;
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "every wavefront loads the same number of rows");
    static_assert(LDS <= 160 * 1024, "");

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

    // Rows [row0, row0 + ROWS) of a panel; rows past the last one are read as the last one (their
    // results are not stored).
    template <int COUNT>
    __device__ static void load_rows(const uint8_t *panel, int rows, int row0, uint8_t *lds)
    {
        const int lane = threadIdx.x & 63, wave = tile_wave();
        const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
        for (int q = 0; q < COUNT / (8 * WAVES); q++) {
            const int at = (q * WAVES + wave) * 8;
            const int row = min(row0 + at + (lane >> 3), rows - 1);
            tile_load16(panel + (int64_t)row * PANEL_BYTES + piece, lds + at * PANEL_BYTES);
        }
    }
    // The scales of those rows, two rows per lane; by the wavefronts from `first` on.
    template <int COUNT>
    __device__ static void load_scales(const uint8_t *scales, int rows, int row0, uint8_t *lds, int first)
    {
        const int lane = threadIdx.x & 63, wave = tile_wave() - first;
        constexpr int PIECES = (COUNT * 8 + 1023) / 1024;
        if (wave >= 0 && wave < PIECES) {
            const int pair = min((row0 >> 1) + wave * 64 + lane, ((rows + 1) >> 1) - 1);
            tile_load16(scales + (int64_t)pair * 16, lds + wave * 1024);
        }
    }
    template <class P>
    __device__ static void load(const P &p, int s, int row0, int col0, uint8_t *buf)
    {
        const TilePanels at = p.at(s);
        load_rows<BM>(at.a, p.a_rows(), row0, buf);
        load_rows<BN>(at.b, p.b_rows(), col0, buf + BM * PANEL_BYTES);
        if (FP4) {
            uint8_t *sc = buf + (BM + BN) * PANEL_BYTES;
            load_scales<BM>(at.a_scales, p.a_rows(), row0, sc, 0);
            load_scales<BN>(at.b_scales, p.b_rows(), col0, sc + SCALES_M, WAVES / 2);
        }
    }

    // acc += the product over panels [s0, s1) of the tile at (row0, col0).  Every wavefront of the
    // workgroup calls it with the same arguments.
    template <class P>
    __device__ void multiply(const P &p, int s0, int s1, int row0, int col0, uint8_t *lds)
    {
        if (s0 >= s1) return;
        const int lane = threadIdx.x & 63, wave = tile_wave();
        const int wm = wave / WGN * WM, wn = wave % WGN * WN;
        const int in_row = lane & 31, half = lane >> 5;
        int place[4];
#pragma unroll
        for (int q = 0; q < 4; q++) place[q] = ((2 * q + half) ^ (lane & 7)) * 16;
        const int a_at = (wm + in_row) * PANEL_BYTES, b_at = (BM + wn + in_row) * PANEL_BYTES;

        load(p, s0, row0, col0, lds);
        int cur = 0;
        for (int s = s0; s < s1; s++) {
            __syncthreads();  // panel s has landed; nobody reads the other buffer any more
            if (s + 1 < s1) load(p, s + 1, row0, col0, lds + (cur ^ BUFFER));
            const uint8_t *buf = lds + cur;
            uint32_t sa[TM][2], sb[TN][2];
            if (FP4) {
                const uint8_t *sc = buf + (BM + BN) * PANEL_BYTES;
#pragma unroll
                for (int i = 0; i < TM; i++) {  // the lane's half of every slice: bytes 0 and 2 of both words
                    const uint64_t v = *(const uint64_t *)(sc + (wm + 32 * i + in_row) * 8) >> (8 * half);
                    sa[i][0] = (uint32_t)v, sa[i][1] = (uint32_t)(v >> 32);
                }
#pragma unroll
                for (int j = 0; j < TN; j++) {
                    const uint64_t v = *(const uint64_t *)(sc + SCALES_M + (wn + 32 * j + in_row) * 8) >> (8 * half);
                    sb[j][0] = (uint32_t)v, sb[j][1] = (uint32_t)(v >> 32);
                }
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                tile_i4 fa[TM], fb[TN];
#pragma unroll
                for (int i = 0; i < TM; i++) fa[i] = *(const tile_i4 *)(buf + a_at + 32 * i * PANEL_BYTES + place[q]);
#pragma unroll
                for (int j = 0; j < TN; j++) fb[j] = *(const tile_i4 *)(buf + b_at + 32 * j * PANEL_BYTES + place[q]);
#pragma unroll
                for (int i = 0; i < TM; i++)
#pragma unroll
                    for (int j = 0; j < TN; j++) acc[i][j] = one(fa[i], fb[j], acc[i][j], q, sa[i], sb[j]);
            }
            cur ^= BUFFER;
        }
        __syncthreads();  // the buffers may be used again
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

    // f(strip, row, col) for every 32 x WN values of the wavefront, strip[r * PITCH + c] in LDS being
    // C[row + r][col + c].  The accumulators hold single rows of 32 columns over half a wavefront;
    // from the strip every lane takes what makes whole 16 bytes of the result.
    template <class F>
    __device__ void store_strips(int row0, int col0, uint8_t *lds, F f)
    {
        const int lane = threadIdx.x & 63, wave = tile_wave();
        const int wm = wave / WGN * WM, wn = wave % WGN * WN;
        float *strip = (float *)lds + wave * 32 * PITCH;
#pragma unroll
        for (int i = 0; i < TM; i++) {
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    strip[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * PITCH + 32 * j + (lane & 31)] = acc[i][j][r];
            wave_fence();
            f(strip, row0 + wm + 32 * i, col0 + wn);
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

// Piece -> (row tile, column tile): bands of 8 row tiles, column by column inside a band, so that
// the ~32 tiles that run on an XCD at once share 8 row tiles and 4 column tiles.
__device__ static inline void tile_place(int piece, int tiles_m, int tiles_n, int *tm, int *tn)
{
    const int band = piece / (8 * tiles_n), first = band * 8, height = min(8, tiles_m - first);
    const int in = piece - band * 8 * tiles_n;
    *tn = in / height;
    *tm = first + in % height;
}
