// Stable sort of n whole numbers below `classes`, least digit first, up to 8 bits a pass.
//
// A wavefront ranks 64 numbers at once: a ballot for each bit of the digit tells every lane who has the same
// digit, the lanes below it among them are its rank, and a counter in LDS for each wavefront and digit goes on from one 64 to the
// next.  The counters' prefix sums in the order (digit, wavefront) are the places.  Nothing is added with
// atomics whose order could show: equal numbers keep their order.
//
// Up to 16384 numbers stay in one workgroup's registers and LDS for all passes: one launch (times below).  More
// go over two launches a pass, tiles of 8192: counts, then places.
#include "tftq_sort.h"

DEV u32 sort_key(const SortArgs &a, int64_t i)
{
    const int64_t id = a.wide ? as_global<const int64_t>(a.ids)[i] : as_global<const int32_t>(a.ids)[i];
    return (uint64_t)id < a.classes && (u32)id != a.skip ? (u32)id : a.classes;
}

// The rank of every item among those of its digit in the wavefront's part, in the order of i, then lanes; `mine` ends
// with how many of every digit there are.
template <int ITEMS>
DEV void sort_rank(const u32 (&digit)[ITEMS], const bool (&live)[ITEMS], int width, u32 *mine, u32 (&rank)[ITEMS])
{
    const uint64_t below = ((uint64_t)1 << (threadIdx.x & 63)) - 1;
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        uint64_t same = __ballot(live[i]);
        for (int b = 0; b < width; b++) {
            const bool bit = digit[i] >> b & 1;
            const uint64_t with = __ballot(bit);
            same &= bit ? with : ~with;
        }
        rank[i] = 0;
        if (live[i]) {
            const u32 before = __builtin_popcountll(same & below), base = mine[digit[i]];
            rank[i] = base + before;
            // every lane has read its counter before the first of its digit moves it on: one wavefront, in order
            __builtin_amdgcn_wave_barrier();
            if (before == 0) mine[digit[i]] = base + (u32)__builtin_popcountll(same);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Exclusive prefix sums of the counters in the order (digit, wavefront), in place; 256 digits.  sums: a u32 a wavefront.
template <int THREADS>
DEV void sort_scan(u32 (*counts)[256], u32 *sums)
{
    constexpr int Q = THREADS / 256;  // threads a digit, four wavefronts' counters to each
    const int digit = threadIdx.x / Q, q = threadIdx.x % Q * 4, lane = threadIdx.x & 63;
    u32 c[4], s = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        c[i] = counts[q + i][digit];
        s += c[i];
    }
    u32 up = s;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u32 from = (u32)__shfl_up((int)up, d);
        if (lane >= d) up += from;
    }
    if (lane == 63) sums[threadIdx.x / 64] = up;
    __syncthreads();
    u32 base = up - s;
    for (int w = 0; w < (int)threadIdx.x / 64; w++) base += sums[w];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        counts[q + i][digit] = base;
        base += c[i];
    }
    __syncthreads();
}

// n numbers in one workgroup, wavefront w the w-th share of 64 ITEMS.
template <int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void k_sort_one(const SortArgs a, int passes, int width)
{
    constexpr int WAVES = THREADS / 64, MOST = THREADS * ITEMS;
    __shared__ u32 counts[WAVES][256], sums[WAVES], keys[MOST];
    __shared__ uint16_t places[MOST];
    const int n = (int)a.n, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    u32 key[ITEMS], place[ITEMS], digit[ITEMS], rank[ITEMS];
    bool live[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        place[i] = (u32)(wave * 64 * ITEMS + i * 64 + lane);
        live[i] = (int)place[i] < n;
        key[i] = live[i] ? sort_key(a, place[i]) : 0;
    }
    for (int pass = 0; pass < passes; pass++) {
        for (int c = threadIdx.x; c < WAVES * 256; c += THREADS) (&counts[0][0])[c] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; i++) digit[i] = key[i] >> (pass * width) & ((1u << width) - 1);
        sort_rank<ITEMS>(digit, live, width, counts[wave], rank);
        __syncthreads();
        sort_scan<THREADS>(counts, sums);
#pragma unroll
        for (int i = 0; i < ITEMS; i++)
            if (live[i]) {
                const u32 to = counts[wave][digit[i]] + rank[i];
                keys[to] = key[i];
                places[to] = (uint16_t)place[i];
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int at = wave * 64 * ITEMS + i * 64 + lane;
            if (live[i]) {
                key[i] = keys[at];
                place[i] = places[at];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int at = wave * 64 * ITEMS + i * 64 + lane;
        if (!live[i]) continue;
        if (a.keys) as_global<u32>(a.keys)[at] = key[i];
        as_global<u32>(a.order)[at] = place[i];
        if (a.position) as_global<u32>(a.position)[place[i]] = (u32)at;
    }
    if (a.offsets)
        for (int64_t c = threadIdx.x; c <= (int64_t)a.classes; c += THREADS)
            as_global<u32>(a.offsets)[c] = (u32)first_at((const u32 *)keys, n, (u32)c);
}

constexpr int SORT_ITEMS = 8, SORT_TILE = 1024 * SORT_ITEMS, SORT_ONE = 16384;

// A pass over many numbers: from ids (the first) or from keys and places.
struct SortPass {
    uint64_t keys, places;  // 0: the ids themselves
    uint64_t to_keys, to_places, position;
    uint64_t counts;        // u32 [tiles][256]
    int shift, width, tiles;
};

DEV u32 sort_read(const SortArgs &a, const SortPass &p, int64_t i) { return p.keys ? as_global<const u32>(p.keys)[i] : sort_key(a, i); }

__global__ __launch_bounds__(1024) void k_sort_count(const SortArgs a, const SortPass p)
{
    __shared__ u32 counts[256];
    if (threadIdx.x < 256) counts[threadIdx.x] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * SORT_TILE;
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++) {
        const int64_t at = first + i * 1024 + threadIdx.x;
        if (at < a.n) atomicAdd(&counts[sort_read(a, p, at) >> p.shift & ((1u << p.width) - 1)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 256) as_global<u32>(p.counts)[(int64_t)blockIdx.x * 256 + threadIdx.x] = counts[threadIdx.x];
}

__global__ __launch_bounds__(1024) void k_sort_place(const SortArgs a, const SortPass p)
{
    __shared__ u32 counts[16][256], sums[16], before[4][256], total[4][256], start[256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, d = threadIdx.x & 255, q = threadIdx.x >> 8;
    for (int c = threadIdx.x; c < 16 * 256; c += 1024) (&counts[0][0])[c] = 0;
    // of digit d: how many there are in all tiles, and in those before this one
    u32 b = 0, t = 0;
    for (int tile = q; tile < p.tiles; tile += 4) {
        const u32 c = as_global<const u32>(p.counts)[(int64_t)tile * 256 + d];
        t += c;
        if (tile < (int)blockIdx.x) b += c;
    }
    before[q][d] = b;
    total[q][d] = t;
    __syncthreads();
    u32 up = 0, own = 0;
    if (threadIdx.x < 256) {
        own = total[0][d] + total[1][d] + total[2][d] + total[3][d];
        up = own;
#pragma unroll
        for (int s = 1; s < 64; s *= 2) {
            const u32 from = (u32)__shfl_up((int)up, s);
            if (lane >= s) up += from;
        }
        if (lane == 63) sums[wave] = up;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
        u32 base = up - own;
        for (int w = 0; w < wave; w++) base += sums[w];
        start[d] = base + before[0][d] + before[1][d] + before[2][d] + before[3][d];
    }
    u32 key[SORT_ITEMS], digit[SORT_ITEMS], rank[SORT_ITEMS], place[SORT_ITEMS];
    bool live[SORT_ITEMS];
    const int64_t first = (int64_t)blockIdx.x * SORT_TILE + wave * 64 * SORT_ITEMS;
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++) {
        const int64_t at = first + i * 64 + lane;
        live[i] = at < a.n;
        key[i] = live[i] ? sort_read(a, p, at) : 0;
        place[i] = live[i] && p.keys ? as_global<const u32>(p.places)[at] : (u32)at;
        digit[i] = key[i] >> p.shift & ((1u << p.width) - 1);
    }
    sort_rank<SORT_ITEMS>(digit, live, p.width, counts[wave], rank);
    __syncthreads();
    // of every wavefront and digit: how many there are in the wavefronts before
    if (threadIdx.x < 256) {
        u32 s = start[d];
        for (int w = 0; w < 16; w++) {
            const u32 c = counts[w][d];
            counts[w][d] = s;
            s += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++) {
        if (!live[i]) continue;
        const u32 to = counts[wave][digit[i]] + rank[i];
        if (p.to_keys) as_global<u32>(p.to_keys)[to] = key[i];
        as_global<u32>(p.to_places)[to] = place[i];
        if (p.position) as_global<u32>(p.position)[place[i]] = to;
    }
}

__global__ __launch_bounds__(256) void k_sort_offsets(const SortArgs a)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c <= (int64_t)a.classes) as_global<u32>(a.offsets)[c] = (u32)first_at(as_global<const u32>(a.keys), a.n, (u32)c);
}

static int sort_passes(int64_t classes)  // numbers from 0 to classes
{
    int bits = 1;
    while (classes >> bits) bits++;
    return bits;
}

int64_t sort_workspace(int64_t n, int64_t classes)
{
    if (n <= SORT_ONE) return 0;
    const int64_t tiles = (n + SORT_TILE - 1) / SORT_TILE, pairs = (sort_passes(classes) + 7) / 8 - 1;
    return tiles * 1024 + std::min<int64_t>(pairs, 2) * ((n * 8 + 15) & ~(int64_t)15);
}

int sort_numbers(const SortArgs &in, void *workspace, hipStream_t st)
{
    SortArgs a = in;
    const int bits = sort_passes(a.classes);
    int passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
    if (a.n <= SORT_ONE) {
        void *args[] = {(void *)&a, (void *)&passes, (void *)&width};
        const void *k = a.n <= 256 ? (const void *)k_sort_one<256, 1> : a.n <= 4096 ? (const void *)k_sort_one<1024, 4> : (const void *)k_sort_one<1024, 16>;
        return (int)hipLaunchKernel(k, dim3(1), dim3(a.n <= 256 ? 256 : 1024), args, 0, st);
    }
    SortPass p = {};
    p.tiles = (int)((a.n + SORT_TILE - 1) / SORT_TILE);
    p.counts = (uint64_t)workspace;
    const uint64_t pairs = p.counts + (uint64_t)p.tiles * 1024, pair = ((uint64_t)a.n * 8 + 15) & ~(uint64_t)15;
    for (int pass = 0; pass < passes; pass++) {
        const bool last = pass == passes - 1;
        p.keys = p.to_keys;
        p.places = p.to_places;
        p.to_keys = last ? a.keys : pairs + (uint64_t)(pass & 1) * pair;
        p.to_places = last ? a.order : p.to_keys + (uint64_t)a.n * 4;
        p.position = last ? a.position : 0;
        p.shift = pass * width;
        p.width = width;
        void *args[] = {(void *)&a, (void *)&p};
        if (const int rc = (int)hipLaunchKernel((const void *)k_sort_count, dim3((unsigned)p.tiles), dim3(1024), args, 0, st)) return rc;
        if (const int rc = (int)hipLaunchKernel((const void *)k_sort_place, dim3((unsigned)p.tiles), dim3(1024), args, 0, st)) return rc;
    }
    if (!a.offsets) return 0;
    void *args[] = {(void *)&a};
    return (int)hipLaunchKernel((const void *)k_sort_offsets, dim3((unsigned)(a.classes / 256 + 1)), dim3(256), args, 0, st);
}
