// Finding the rank-th highest of many floats by counting: on integers that are ordered as the
// floats are, because floats themselves may be too close to divide their range (halves and
// quotients of numbers below the normal range round, and a range that does not shrink is a
// loop that does not end).  Plain C++ (no CUDA headers needed), so that a host-only test can
// drive it over such numbers.
#pragma once

#include <stdint.h>
#include <string.h>

#ifndef NB200_HD
#ifdef __CUDACC__
#define NB200_HD __host__ __device__ __forceinline__
#else
#define NB200_HD inline
#endif
#endif

namespace nb200 {

// Order-preserving map of a float that is not NaN; both zeros have one key.
NB200_HD uint32_t score_key32(float s)
{
    s += 0.0f;                                   // -0 -> +0
    uint32_t u;
    memcpy(&u, &s, 4);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

NB200_HD float score_of_key(uint32_t key)
{
    const uint32_t u = (key >> 31) ? key & 0x7FFFFFFFu : ~key;
    float s;
    memcpy(&s, &u, 4);
    return s;
}

// Keys low .. high and their division into at most 256 bins of 2^shift keys.  With low < high
// the two ends lie in different bins, and a bin's range is at most 1/128 of the whole: 32 bits
// are used up after five rounds at most, the last one with bins of a single key.
struct RankRange
{
    uint32_t low, high;
    int shift;
};

NB200_HD RankRange rank_range(uint32_t low, uint32_t high)
{
    RankRange r = {low, high, 0};
    while((high - low) >> r.shift > 255u)
    {
        ++r.shift;
    }
    return r;
}

NB200_HD bool rank_inside(const RankRange &r, uint32_t key)
{
    return key >= r.low && key <= r.high;
}

NB200_HD int rank_bin(const RankRange &r, uint32_t key)
{
    return (int)((key - r.low) >> r.shift);
}

// The keys of bin `bin`, which are the range of the next round.
NB200_HD RankRange rank_narrowed(const RankRange &r, int bin)
{
    const uint32_t low = r.low + ((uint32_t)bin << r.shift);
    const uint32_t last = ((uint32_t)1 << r.shift) - 1u;
    return rank_range(low, r.high - low < last ? r.high : low + last);
}

} // namespace nb200
