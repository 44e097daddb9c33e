// Stable sort of n whole numbers below `classes`, least digit first.
//
// A wavefront ranks 64 numbers at once: a ballot for each bit of the digit tells every lane who has the same
// digit, the lanes below it among them are its rank, and a counter in LDS for each wavefront and digit goes on from one
// 64 to the next.  The counters' prefix sums in the order (digit, wavefront) are the places.  Nothing is added
// with atomics whose order could show: equal numbers keep their order.
//
// Few numbers stay in one workgroup's registers and LDS for all passes of up to 9 bits: one launch, bound by the four
// vector units of one compute unit (four instructions a bit and number).  More go over two launches a pass of as many
// bits: counts of tiles of 2048, then places (three from 131072 on, where every tile would read too many counts).  Numbers
// that another stream changes between the two would not fit the counts; places are held below n, whatever memory says.
#include "tftq_sort.h"
#include "tftq_fill.h"

DEV u32 sort_key(const SortArgs &a, int64_t i)
{
    const int64_t id = a.wide ? as_global<const int64_t>(a.ids)[i] : as_global<const int32_t>(a.ids)[i];
    return (uint64_t)id < a.classes && (u32)id != a.skip ? (u32)id : a.classes;
}

// What the wavefront's lanes wrote to LDS is there for all of them; nothing to wait for, as one wavefront's accesses stay in order.
DEV void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The rank of every item among those of its digit in the wavefront's part, in the order of i, then lanes; `mine`, this
// wavefront's counters, ends with how many of every digit there are.  Items from `items` on are not live.
template <int ITEMS>
DEV void sort_rank(const u32 (&digit)[ITEMS], const bool (&live)[ITEMS], int items, int width, u32 *mine, u32 (&rank)[ITEMS])
{
    u32 low[ITEMS], high[ITEMS];  // who has the same digit
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const uint64_t all = __ballot(live[i]);
        low[i] = (u32)all;
        high[i] = (u32)(all >> 32);
    }
    for (int b = 0; b < width; b++) {
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            if (ITEMS > 4 && i >= items) continue;
            const u32 mask = (u32)((int)(digit[i] << (31 - b)) >> 31);
            const uint64_t with = __ballot(mask != 0);
            low[i] &= ~((u32)with ^ mask);
            high[i] &= ~((u32)(with >> 32) ^ mask);
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        rank[i] = 0;
        if (live[i]) {
            const u32 before = __builtin_amdgcn_mbcnt_hi(high[i], __builtin_amdgcn_mbcnt_lo(low[i], 0)), base = mine[digit[i]];
            rank[i] = base + before;
            // every lane has read its counter before the first of its digit moves it on, and the next item's read is behind that
            wave_sync();
            if (before == 0) mine[digit[i]] = base + (u32)(__builtin_popcount(low[i]) + __builtin_popcount(high[i]));
            wave_sync();
        }
    }
}

// The exclusive prefix sum of v over the workgroup's threads; sums: a u32 a wavefront, free again behind the next barrier.
DEV u32 sort_prefix(u32 v, u32 *sums)
{
    u32 up = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u32 from = (u32)__shfl_up((int)up, d);
        if ((int)(threadIdx.x & 63) >= d) up += from;
    }
    if ((threadIdx.x & 63) == 63) sums[threadIdx.x / 64] = up;
    __syncthreads();
    u32 base = up - v;
    for (int w = 0; w < (int)threadIdx.x / 64; w++) base += sums[w];
    return base;
}

// Workgroups from `tiles` on write zeros, a vector to a lane: they start and end in their order, so that what is written at
// a time is one piece of memory that moves on (1050 MB at 6.6 TB/s; 5.3 with 64 KB to a workgroup, 4.7 with as many
// workgroups as run at once and all of them side by side).
template <int THREADS>
DEV bool sort_fill(const SortArgs &a, int tiles)
{
    if ((int)blockIdx.x < tiles) return false;
    const int rounds = fill_rounds(a.fill_bytes);
    int64_t at = ((int64_t)((int)blockIdx.x - tiles) * rounds * THREADS + threadIdx.x) * 16;
    for (int r = 0; r < rounds; r++, at += THREADS * 16)
        if (at < a.fill_bytes) store_bytes(a.fill + (uint64_t)at, (u32)min((int64_t)16, a.fill_bytes - at), u32x4{0, 0, 0, 0});
    return true;
}

// n numbers in one workgroup, wavefront w the w-th share of them.
template <int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void k_sort_one(const SortArgs a, int passes, int width)
{
    constexpr int WAVES = THREADS / 64, MOST = THREADS * ITEMS, DIGITS = THREADS == 256 ? 256 : 512;
    constexpr int Q = THREADS / DIGITS, EACH = WAVES / Q;  // threads to a digit, wavefronts' counters to a thread
    __shared__ u32 counts[WAVES][DIGITS], sums[WAVES], keys[MOST];
    __shared__ uint16_t places[MOST];
    if (sort_fill<THREADS>(a, 1)) return;
    const int n = (int)a.n, lane = threadIdx.x & 63, items = (n + THREADS - 1) / THREADS, first = (int)(threadIdx.x / 64) * 64 * items + lane;
    u32 *mine = counts[threadIdx.x / 64];
    u32 key[ITEMS], place[ITEMS], digit[ITEMS], rank[ITEMS];
    bool live[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        place[i] = (u32)(first + i * 64);
        live[i] = i < items && (int)place[i] < n;
        key[i] = live[i] ? sort_key(a, place[i]) : 0;
    }
    for (int pass = 0; pass < passes; pass++) {
        for (int c = threadIdx.x; c < WAVES * DIGITS; c += THREADS) (&counts[0][0])[c] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; i++) digit[i] = key[i] >> (pass * width) & ((1u << width) - 1);
        sort_rank<ITEMS>(digit, live, items, width, mine, rank);
        __syncthreads();
        {
            const int d = threadIdx.x / Q, w = threadIdx.x % Q * EACH;
            u32 c[EACH], s = 0;
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                c[i] = counts[w + i][d];
                s += c[i];
            }
            u32 base = sort_prefix(s, sums);
#pragma unroll
            for (int i = 0; i < EACH; i++) {
                counts[w + i][d] = base;
                base += c[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; i++)
            if (live[i]) {
                const u32 to = mine[digit[i]] + rank[i];
                keys[to] = key[i];
                places[to] = (uint16_t)place[i];
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; i++)
            if (live[i]) {
                key[i] = keys[first + i * 64];
                place[i] = places[first + i * 64];
            }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        if (!live[i]) continue;
        const int at = first + i * 64;
        if (a.keys) as_global<u32>(a.keys)[at] = key[i];
        as_global<u32>(a.order)[at] = place[i];
        if (a.position) as_global<u32>(a.position)[place[i]] = (u32)at;
    }
    if (a.offsets)
        for (int64_t c = threadIdx.x; c <= (int64_t)a.classes; c += THREADS)
            as_global<u32>(a.offsets)[c] = (u32)first_at((const u32 *)keys, n, c);
}

constexpr int SORT_THREADS = 512, SORT_ITEMS = 4, SORT_TILE = SORT_THREADS * SORT_ITEMS, SORT_DIGITS = 512;
constexpr int SORT_DIRECT = 64;  // so many tiles read each other's counts themselves

// A pass over many numbers: from ids (the first) or from keys and places.
struct SortPass {
    uint64_t keys, places;  // 0: the ids themselves
    uint64_t to_keys, to_places, position, offsets;
    uint64_t counts;        // u32 [SORT_DIGITS][pitch]: of a digit and a tile; with more than SORT_DIRECT tiles, then u32 [SORT_DIGITS] of all
    int shift, width, tiles, pitch;
};

DEV u32 sort_read(const SortArgs &a, const SortPass &p, int64_t i) { return p.keys ? as_global<const u32>(p.keys)[i] : sort_key(a, i); }

__global__ __launch_bounds__(SORT_THREADS) void k_sort_count(const SortArgs a, const SortPass p)
{
    __shared__ u32 counts[SORT_DIGITS];
    if (sort_fill<SORT_THREADS>(a, p.tiles)) return;
    counts[threadIdx.x] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * SORT_TILE + threadIdx.x;
    u32 key[SORT_ITEMS];
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++) key[i] = first + i * SORT_THREADS < a.n ? sort_read(a, p, first + i * SORT_THREADS) : 0;
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++)
        if (first + i * SORT_THREADS < a.n) atomicAdd(&counts[key[i] >> p.shift & ((1u << p.width) - 1)], 1u);
    __syncthreads();
    if (threadIdx.x >> p.width == 0) as_global<u32>(p.counts)[(int64_t)threadIdx.x * p.pitch + blockIdx.x] = counts[threadIdx.x];
}

// A workgroup to a digit: its counts become how many there are in the tiles before.
__global__ __launch_bounds__(256) void k_sort_before(const SortPass p)
{
    __shared__ u32 sums[4];
    GLOBAL u32 *row = as_global<u32>(p.counts) + (int64_t)blockIdx.x * p.pitch;
    u32 base = 0;
    for (int tile = 0; tile < p.tiles; tile += 256) {
        const int at = tile + (int)threadIdx.x;
        const u32 c = at < p.tiles ? row[at] : 0, before = sort_prefix(c, sums);
        if (at < p.tiles) row[at] = base + before;
        base += sums[0] + sums[1] + sums[2] + sums[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) as_global<u32>(p.counts)[(int64_t)SORT_DIGITS * p.pitch + blockIdx.x] = base;
}

__global__ __launch_bounds__(SORT_THREADS) void k_sort_place(const SortArgs a, const SortPass p)
{
    constexpr int WAVES = SORT_THREADS / 64;
    __shared__ u32 counts[WAVES][SORT_DIGITS], sums[WAVES];
    if (sort_fill<SORT_THREADS>(a, p.tiles)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, d = threadIdx.x;
    u32 key[SORT_ITEMS], digit[SORT_ITEMS], rank[SORT_ITEMS], place[SORT_ITEMS];
    bool live[SORT_ITEMS];
    const int64_t first = (int64_t)blockIdx.x * SORT_TILE + wave * 64 * SORT_ITEMS + lane;
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++) {
        const int64_t at = first + i * 64;
        live[i] = at < a.n;
        key[i] = live[i] ? sort_read(a, p, at) : 0;
        place[i] = live[i] && p.keys ? min(as_global<const u32>(p.places)[at], (u32)a.n - 1) : (u32)at;
    }
    // of digit d: how many there are in all tiles, and in those before this one
    u32 before = 0, total = 0;
    if (d >> p.width == 0) {
        if (p.tiles > SORT_DIRECT) {
            before = as_global<const u32>(p.counts)[(int64_t)d * p.pitch + blockIdx.x];
            total = as_global<const u32>(p.counts)[(int64_t)SORT_DIGITS * p.pitch + d];
        } else {
            for (int tile = 0; tile < p.tiles; tile += 4) {
                const u32x4 c = *(as_global<const u32x4>(p.counts + ((uint64_t)d * p.pitch + tile) * 4));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (tile + i >= p.tiles) continue;
                    total += c[i];
                    if (tile + i < (int)blockIdx.x) before += c[i];
                }
            }
        }
    }
#pragma unroll
    for (int w = 0; w < WAVES; w++) counts[w][d] = 0;
    const u32 start = sort_prefix(total, sums);  // a barrier
    if (p.offsets && blockIdx.x == 0 && d <= (int)a.classes) as_global<u32>(p.offsets)[d] = start;
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++) digit[i] = key[i] >> p.shift & ((1u << p.width) - 1);
    sort_rank<SORT_ITEMS>(digit, live, SORT_ITEMS, p.width, counts[wave], rank);
    __syncthreads();
    u32 s = start + before;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        const u32 c = counts[w][d];
        counts[w][d] = s;
        s += c;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SORT_ITEMS; i++) {
        if (!live[i]) continue;
        const u32 to = min(counts[wave][digit[i]] + rank[i], (u32)a.n - 1);
        if (p.to_keys) as_global<u32>(p.to_keys)[to] = key[i];
        as_global<u32>(p.to_places)[to] = place[i];
        if (p.position) as_global<u32>(p.position)[place[i]] = to;
    }
}

__global__ __launch_bounds__(256) void k_sort_offsets(const SortArgs a)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c <= (int64_t)a.classes) as_global<u32>(a.offsets)[c] = (u32)first_at(as_global<const u32>(a.keys), a.n, c);
}

static int sort_bits(int64_t classes)  // numbers from 0 to classes
{
    int bits = 1;
    while (classes >> bits) bits++;
    return bits;
}

// Whether one workgroup takes all.  Times of a sort with places and offsets, us, in one workgroup and in tiles:
// 4096 numbers below 8 6.5, 7.2, below 255 7.7, 7.5, below 1000 11.1, 18.4; 8192 9.3, 7.3 / 13.0, 8.0 / 17.7, 19.4; 16384
// 16.3, 7.6 / 23.7, 8.5 / 31.1, 20.6: one compute unit's scattered stores, and its ballots, against two launches a pass.
static bool sort_one(int64_t n, int64_t classes) { return n <= (classes >= SORT_DIGITS ? 8192 : 4096); }

// Whether the offsets are a launch of their own, which searches the keys: a tile that knows all digits' places writes
// them along with a sort of one pass, and one workgroup up to 2048.
static bool sort_searches(int64_t n, int64_t classes) { return classes >= (sort_one(n, classes) ? 2049 : SORT_DIGITS); }

static int64_t sort_pitch(int64_t n) { return ((n + SORT_TILE - 1) / SORT_TILE + 3) & ~(int64_t)3; }

int64_t sort_workspace(int64_t n, int64_t classes)
{
    if (sort_one(n, classes)) return 0;
    const int64_t pairs = (sort_bits(classes) + 8) / 9 - 1;
    return (sort_pitch(n) + 1) * SORT_DIGITS * 4 + std::min<int64_t>(pairs, 2) * ((n * 8 + 15) & ~(int64_t)15);
}

bool sort_needs_keys(int64_t n, int64_t classes) { return sort_searches(n, classes); }

// Workgroups for so many tiles and the zeros.
static unsigned sort_groups(const SortArgs &a, int tiles, int threads)
{
    return (unsigned)(tiles + fill_groups(a.fill_bytes, threads));
}

static int sort_offsets(SortArgs a, hipStream_t st)
{
    void *args[] = {(void *)&a};
    return (int)hipLaunchKernel((const void *)k_sort_offsets, dim3((unsigned)(a.classes / 256 + 1)), dim3(256), args, 0, st);
}

int sort_numbers(const SortArgs &in, void *workspace, hipStream_t st)
{
    SortArgs a = in;
    const int bits = sort_bits(a.classes);
    if (sort_one(a.n, a.classes)) {
        const int most = a.n <= 256 ? 8 : 9;
        int passes = (bits + most - 1) / most, width = (bits + passes - 1) / passes;
        void *args[] = {(void *)&a, (void *)&passes, (void *)&width};
        const void *k = a.n <= 256    ? (const void *)k_sort_one<256, 1>
                        : a.n <= 4096 ? (const void *)k_sort_one<1024, 4>
                                      : (const void *)k_sort_one<1024, 8>;
        const uint64_t offsets = a.offsets;
        if (sort_searches(a.n, a.classes)) a.offsets = 0;
        const int rc = (int)hipLaunchKernel(k, dim3(sort_groups(a, 1, a.n <= 256 ? 256 : 1024)), dim3(a.n <= 256 ? 256 : 1024), args, 0, st);
        if (rc || a.offsets == offsets) return rc;
        a.offsets = offsets;
        return sort_offsets(a, st);
    }
    const int passes = (bits + 8) / 9, width = (bits + passes - 1) / passes;
    SortPass p = {};
    p.tiles = (int)((a.n + SORT_TILE - 1) / SORT_TILE);
    p.pitch = (int)sort_pitch(a.n);
    p.counts = (uint64_t)workspace;
    p.width = width;
    const uint64_t pairs = p.counts + (uint64_t)(p.pitch + 1) * SORT_DIGITS * 4, pair = ((uint64_t)a.n * 8 + 15) & ~(uint64_t)15;
    int launch = 0;
    auto next_share = [&] {  // of the zeros
        const int64_t begin = fill_begin(in.fill_bytes, 2 * passes, launch++);
        a.fill = in.fill + (uint64_t)begin;
        a.fill_bytes = fill_begin(in.fill_bytes, 2 * passes, launch) - begin;
    };
    for (int pass = 0; pass < passes; pass++) {
        const bool last = pass == passes - 1;
        p.keys = p.to_keys;
        p.places = p.to_places;
        p.to_keys = last ? a.keys : pairs + (uint64_t)(pass & 1) * pair;
        p.to_places = last ? a.order : p.to_keys + (uint64_t)a.n * 4;
        p.position = last ? a.position : 0;
        p.offsets = passes == 1 ? a.offsets : 0;
        p.shift = pass * width;
        void *args[] = {(void *)&a, (void *)&p}, *before[] = {(void *)&p};
        next_share();
        if (const int rc = (int)hipLaunchKernel((const void *)k_sort_count, dim3(sort_groups(a, p.tiles, SORT_THREADS)), dim3(SORT_THREADS), args, 0, st)) return rc;
        if (p.tiles > SORT_DIRECT)
            if (const int rc = (int)hipLaunchKernel((const void *)k_sort_before, dim3(1u << width), dim3(256), before, 0, st)) return rc;
        next_share();
        if (const int rc = (int)hipLaunchKernel((const void *)k_sort_place, dim3(sort_groups(a, p.tiles, SORT_THREADS)), dim3(SORT_THREADS), args, 0, st)) return rc;
    }
    return a.offsets && passes > 1 ? sort_offsets(a, st) : 0;
}
