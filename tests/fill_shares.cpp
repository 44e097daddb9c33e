// Replays where zeros beside other work are written: `bytes shares threads` lines in, the bytes that no share covers, those
// that two do, and those that its workgroups leave out, out.
#include "../torchft_amd/csrc/tftq_fill.h"

#include <cstdio>

int main()
{
    long long bytes;
    int shares, threads;
    while (std::scanf("%lld %d %d", &bytes, &shares, &threads) == 3) {
        long long missing = 0, twice = 0, left = 0, at = 0;
        for (int i = 0; i < shares; i++) {
            const int64_t begin = fill_begin(bytes, shares, i), share = fill_begin(bytes, shares, i + 1) - begin;
            missing += std::max<long long>(0, begin - at);
            twice += std::max<long long>(0, at - begin) + std::max<long long>(0, -share);
            at = begin + share;
            left += std::max<long long>(0, share - fill_groups(share, threads) * threads * 16 * fill_rounds(share));
        }
        std::printf("%lld %lld %lld\n", missing + bytes - at, twice, left);
    }
}
