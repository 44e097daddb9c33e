// A stable sort of whole numbers, shared by the embedding's gradient and the experts (tftq_sort.hip).
#pragma once

#include "tftq_rows.h"

struct SortArgs {
    uint64_t ids;      // n numbers of `wide` ? 8 : 4 bytes, signed
    int wide;
    int64_t n;
    u32 classes;       // numbers outside [0, classes), and `skip`, count as `classes`, the last
    u32 skip;          // none: classes
    uint64_t keys;     // u32 [n]: the numbers in order; 0: not wanted (sort_needs_keys)
    uint64_t order;    // u32 [n]: where they stood
    uint64_t position; // u32 [n]: where they went; 0: not wanted
    uint64_t offsets;  // u32 [classes + 1]: how many are below 0, 1, ... classes; 0: not wanted
    uint64_t fill;     // fill_bytes of zeros to write on the side: a sort leaves most of the machine idle
    int64_t fill_bytes;
};

__attribute__((visibility("hidden"))) int64_t sort_workspace(int64_t n, int64_t classes);  // bytes, a multiple of 16
// Whether `keys` has to be there for `offsets`.
__attribute__((visibility("hidden"))) bool sort_needs_keys(int64_t n, int64_t classes);
__attribute__((visibility("hidden"))) int sort_numbers(const SortArgs &a, void *workspace, hipStream_t st);

// The first of n ascending keys that is not below k.
template <class P>
DEV int64_t first_at(P keys, int64_t n, int64_t k)
{
    int64_t lo = 0;
    while (n > 0) {
        const int64_t half = n >> 1;
        if (keys[lo + half] < k) {
            lo += half + 1;
            n -= half + 1;
        } else n = half;
    }
    return lo;
}
