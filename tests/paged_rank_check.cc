// Host check of nntile_b200/csrc/paged_rank.hh: the search that the block ranking makes ends,
// and with the right score, also where the scores are numbers below the normal range,
// neighbours, or far apart.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <functional>
#include <random>
#include <vector>

#include "../nntile_b200/csrc/paged_rank.hh"

using namespace nb200;

#define CHECK(x) do { if(!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while(0)

// the kernel's search, its list of candidates left out: until one key is left
static float rank_th(const std::vector<float> &v, int rank, int &rounds)
{
    float low = v[0], high = v[0];
    for(float s : v)
    {
        low = std::min(low, s);
        high = std::max(high, s);
    }
    RankRange r = rank_range(score_key32(low), score_key32(high));
    rounds = 0;
    while(r.low < r.high && rounds < 100)
    {
        int bins[256] = {}, above = 0, bin = 255;
        for(float s : v)
        {
            const uint32_t key = score_key32(s);
            if(rank_inside(r, key))
            {
                if(rank_bin(r, key) < 0 || rank_bin(r, key) > 255) return NAN;
                ++bins[rank_bin(r, key)];
            }
        }
        while(above + bins[bin] < rank)
        {
            above += bins[bin--];
        }
        rank -= above;
        r = rank_narrowed(r, bin);
        ++rounds;
    }
    return score_of_key(r.low);
}

static int check(std::vector<float> v)
{
    std::vector<float> sorted = v;
    std::sort(sorted.begin(), sorted.end(), std::greater<float>());
    for(int rank : {1, 2, (int)v.size()/3 + 1, (int)v.size()/2 + 1, (int)v.size() - 1, (int)v.size()})
    {
        if(rank < 1 || rank > (int)v.size()) continue;
        int rounds;
        const float found = rank_th(v, rank, rounds);
        CHECK(found == sorted[rank - 1]);
        CHECK(rounds <= 5);
    }
    return 0;
}

int main()
{
    const float tiny = std::ldexp(1.0f, -149);
    CHECK(tiny > 0.0f);
    CHECK(score_key32(-0.0f) == score_key32(0.0f));
    const float order[] = {-FLT_MAX, -1.0f, -FLT_MIN, -tiny, 0.0f, tiny, 2*tiny, FLT_MIN, 1.0f, FLT_MAX};
    for(int i = 0; i < 10; ++i)
    {
        CHECK(score_of_key(score_key32(order[i])) == order[i]);
        CHECK(i == 0 || score_key32(order[i - 1]) < score_key32(order[i]));
    }
    for(float base : order)
    {
        // two neighbours, hundreds of each, and a run of neighbours
        const float next = std::nextafter(base, INFINITY);
        std::vector<float> two, run, far;
        float s = base;
        for(int i = 0; i < 300; ++i)
        {
            two.push_back(base);
            two.push_back(std::isfinite(next) ? next : base);
            run.push_back(s);
            run.push_back(s);
            s = std::isfinite(std::nextafter(s, INFINITY)) ? std::nextafter(s, INFINITY) : s;
            far.push_back(i % 3 == 0 ? base : i % 3 == 1 ? -FLT_MAX : FLT_MAX);
        }
        if(check(two) || check(run) || check(far)) return 1;
        if(check(std::vector<float>(400, base)) || check({base}) || check({base, -base})) return 1;
    }
    for(int odd = 2; odd < 12; ++odd)            // halves of odd numbers of the smallest step
    {
        std::vector<float> v;
        for(int i = 0; i < 600; ++i) v.push_back((odd + (i & 1))*tiny);
        if(check(v)) return 1;
    }
    std::mt19937 rng(1);
    for(int t = 0; t < 200; ++t)
    {
        std::vector<float> v;
        const int spread = t % 140;
        for(int i = 0; i < 700; ++i)
        {
            const float x = std::normal_distribution<float>()(rng);
            v.push_back(std::ldexp(x, -spread - (t & 1 ? (int)(rng() % 20) : 0)));
        }
        if(check(v)) return 1;
    }
    return 0;
}
