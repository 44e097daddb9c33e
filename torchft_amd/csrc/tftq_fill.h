// Zeros written beside other work, in shares: a launch's workgroups behind those of its own work write one share, a vector of 16
// bytes to a lane and round.  Host arithmetic without HIP types, so that it can be replayed by a host compiler.
#pragma once

#include "tftq_internal.h"

#include <algorithm>

// Rounds of a workgroup: a grid has fewer than 2^32 threads.
TFTQ_HD static inline int fill_rounds(int64_t bytes) { return (int)(bytes >> 34) + 1; }
// Workgroups of a share.
static inline int64_t fill_groups(int64_t bytes, int threads)
{
    const int64_t each = (int64_t)threads * 16 * fill_rounds(bytes);
    return (bytes + each - 1) / each;
}
// Where the i-th of so many shares begins; the last ends with the bytes.
static inline int64_t fill_begin(int64_t bytes, int shares, int i)
{
    const int64_t share = (bytes / shares + 4095) & ~(int64_t)4095;
    return i == shares ? bytes : std::min(bytes, i * share);
}
