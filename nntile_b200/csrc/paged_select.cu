// Choosing the blocks of a paged cache that a new token attends to.
//
// For query heads q_g (g < group) and the bounds kmin, kmax of a block's stored keys,
//     score = max_g sum_d max(q_gd, 0)*kmax_d + min(q_gd, 0)*kmin_d,
// the least upper bound on q_g.k over every key inside the bounds.  The blocks with the
// highest scores are selected, ties by the lowest index: the answer is a set that must not
// depend on the order of any sum.
//
// Scoring reads 4*head bytes a block and is bound by HBM bandwidth; it runs on the
// warp-level tensor instruction with fp32 sums (q split into its positive and negative part is
// an ordinary product) and keeps a bound of each sum's error beside it.  Ranking then needs
// exact sums only for the blocks within that bound of the last one taken, a handful in
// practice: those are added up again in 64 bits, where products of 16-bit factors are exact.
// The bound: a truncating accumulation of 16 products and the running sum in fp32 loses at
// most 17 units of 2^-23 of the sum of magnitudes a step; head <= 256 takes 32 steps, so
// 32*17*2^-23 < 2^-13 of sum_d |q_d||k_d|, which a second product of magnitudes delivers.
#include <algorithm>

#include "paged.cuh"
#include "per_device.hh"

namespace nb200 {

constexpr float SCORE_ERROR = 1.0f/8192.0f;      // 2^-13
constexpr float SCORE_FLOOR = 1e-30f;            // products below the normal range

// Order-preserving map of a double to an unsigned integer; NaN above everything.
__device__ __forceinline__ unsigned long long score_key(double s)
{
    if(s != s)
    {
        return ~0ull;
    }
    const unsigned long long u = (unsigned long long)__double_as_longlong(s + 0.0);   // -0 -> +0
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
// The same for a float that is not NaN.
__device__ __forceinline__ uint32_t score_key32(float s)
{
    const uint32_t u = __float_as_uint(s + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

struct PagedSelectArgs
{
    int head, page_size, num_pages, max_blocks, batch, group, kv_heads, num_selected;
    int first_blocks, last_blocks;
    const int32_t *lengths, *block_table;
    const void *q, *bounds;
    int32_t *selected;
    float2 *scores;                              // [unit][block]: score, bound of its error
    unsigned long long *keys;                    // [unit][block]: exact, where it was needed
    uint32_t *status;
};

// The exact key of a block, by a whole warp (same value in every lane).
template<typename T>
__device__ __forceinline__ unsigned long long exact_key(const PagedSelectArgs &a, int kvh, int b,
        int page, int lane)
{
    const T *low = (const T *)a.bounds + ((size_t)page*a.kv_heads + kvh)*2*a.head;
    const T *high = low + a.head;
    unsigned long long best = 0ull;
    for(int g = 0; g < a.group; ++g)
    {
        const T *q = (const T *)a.q + (((size_t)kvh*a.group + g)*a.batch + b)*a.head;
        double s = 0.0;
        for(int h = lane; h < a.head; h += 32)
        {
            const double x = (double)to_f(q[h]);
            s += (x > 0.0 ? x : 0.0)*(double)to_f(high[h])
                    + (x < 0.0 ? x : 0.0)*(double)to_f(low[h]);
            if(x != x)
            {
                s = x;
            }
        }
#pragma unroll
        for(int o = 16; o > 0; o >>= 1)
        {
            s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        const unsigned long long key = score_key(s);
        best = key > best ? key : best;
    }
    return best;
}

__device__ __forceinline__ int filled_blocks(const PagedSelectArgs &a, int b, uint32_t *status)
{
    return blocks_of(checked_length(a.lengths, b, a.max_blocks*a.page_size, status), a.page_size);
}

// Any head: a warp per block, sums in 64 bits, rounded once.
template<typename T>
__global__ void __launch_bounds__(128)
paged_score_generic_kernel(const PagedSelectArgs a)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = (a.max_blocks + 3)/4;
    const int unit = blockIdx.x/chunks;
    const int block = (blockIdx.x - unit*chunks)*4 + warp;
    const int b = unit % a.batch, kvh = unit/a.batch;
    if(block >= filled_blocks(a, b, a.status))
    {
        return;
    }
    const int page = checked_page(a.block_table + (size_t)b*a.max_blocks, block, a.num_pages,
            a.status);
    float s = -CUDART_INF_F, error = 0.0f;
    if(page >= 0)
    {
        const unsigned long long key = exact_key<T>(a, kvh, b, page, lane);
        const double exact = __longlong_as_double((long long)((key >> 63)
                ? key & 0x7FFFFFFFFFFFFFFFull : ~key));
        s = key == ~0ull ? CUDART_NAN_F : (float)exact;
        error = fabsf(s)*1.2e-7f + SCORE_FLOOR;          // infinite and NaN ones stay so
    }
    if(lane == 0)
    {
        a.scores[(size_t)unit*a.max_blocks + block] = make_float2(s, error);
    }
}

template<typename T>
__device__ __forceinline__ void score_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
        uint32_t a3, uint32_t b0, uint32_t b1);
template<>
__device__ __forceinline__ void score_mma<bf16>(float (&c)[4], uint32_t a0, uint32_t a1,
        uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template<>
__device__ __forceinline__ void score_mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1,
        uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The positive or the negative halves of a word; NaN stays.
template<typename T, bool POSITIVE>
__device__ __forceinline__ uint32_t half_of(uint32_t w)
{
    const float2 f = unpack2<T>(w);
    return POSITIVE ? pack2<T>(max_nan(f.x, 0.0f), max_nan(f.y, 0.0f))
            : pack2<T>(min_nan(f.x, 0.0f), min_nan(f.y, 0.0f));
}

// A warp scores 8*NT neighbouring blocks of a unit against 16 heads at a time.  The order of
// the head elements is free in a sum, so a lane's 16-byte piece t + 4j of a bounds row is the
// operand of two steps as it comes from memory: no staging, 16 bytes a load, and with
// NT = 2 for heads up to 128 sixteen loads (8 KB a warp) in flight at once.
constexpr int SCORE_WARPS = 4;

template<typename T, int DP, int NT, bool WIDE>
__global__ void __launch_bounds__(SCORE_WARPS*32)
paged_score_kernel(const PagedSelectArgs a)
{
    constexpr int JN = DP/32, PER_CTA = SCORE_WARPS*8*NT;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = lane >> 2, t = lane & 3;
    const int chunks = (a.max_blocks + PER_CTA - 1)/PER_CTA;
    const int unit = blockIdx.x/chunks, chunk = blockIdx.x - unit*chunks;
    const int b = unit % a.batch, kvh = unit/a.batch;
    const int count = filled_blocks(a, b, a.status);
    const int block0 = chunk*PER_CTA + warp*8*NT;
    if(block0 >= count)
    {
        return;
    }
    // bounds of block n of each tile: kmin rows first, then kmax
    uint4 kb[NT][2][JN];
    bool missing[NT];
#pragma unroll
    for(int i = 0; i < NT; ++i)
    {
        const int block = block0 + 8*i + n;
        const int page = block < count ? checked_page(a.block_table + (size_t)b*a.max_blocks,
                block, a.num_pages, a.status) : -1;
        missing[i] = page < 0;
        const T *row = (const T *)a.bounds + ((size_t)max(page, 0)*a.kv_heads + kvh)*2*a.head;
#pragma unroll
        for(int j = 0; j < JN; ++j)
        {
            const int h = 8*(t + 4*j);
            const bool on = page >= 0 && h < a.head;
            kb[i][0][j] = on ? __ldg(reinterpret_cast<const uint4 *>(row + h))
                    : make_uint4(0u, 0u, 0u, 0u);
            kb[i][1][j] = on ? __ldg(reinterpret_cast<const uint4 *>(row + a.head + h))
                    : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    float best[NT][2], error[NT][2];
#pragma unroll
    for(int i = 0; i < NT; ++i)
#pragma unroll
        for(int x = 0; x < 2; ++x)
        {
            best[i][x] = -CUDART_INF_F;
            error[i][x] = 0.0f;
        }
    constexpr int ROWS = WIDE ? 16 : 8;
    for(int g0 = 0; g0 < a.group; g0 += ROWS)
    {
        // s: scores; up, down: sums of magnitudes, of the two halves of q (down is negative)
        float s[NT][4], up[NT][4], down[NT][4];
#pragma unroll
        for(int i = 0; i < NT; ++i)
#pragma unroll
            for(int x = 0; x < 4; ++x)
                s[i][x] = up[i][x] = down[i][x] = 0.0f;
#pragma unroll
        for(int j = 0; j < JN; ++j)
        {
            uint32_t qw[WIDE ? 2 : 1][4];
#pragma unroll
            for(int m = 0; m < (WIDE ? 2 : 1); ++m)
            {
                const int g = g0 + 8*m + n, h = 8*(t + 4*j);
                const uint4 v = g < a.group && h < a.head ? *reinterpret_cast<const uint4 *>(
                        (const T *)a.q + (((size_t)kvh*a.group + g)*a.batch + b)*a.head + h)
                        : make_uint4(0u, 0u, 0u, 0u);
                qw[m][0] = v.x;
                qw[m][1] = v.y;
                qw[m][2] = v.z;
                qw[m][3] = v.w;
            }
#pragma unroll
            for(int w = 0; w < 4; w += 2)
            {
                const uint32_t p0 = half_of<T, true>(qw[0][w]), p2 = half_of<T, true>(qw[0][w + 1]);
                const uint32_t m0 = half_of<T, false>(qw[0][w]),
                        m2 = half_of<T, false>(qw[0][w + 1]);
                uint32_t p1 = 0u, p3 = 0u, m1 = 0u, m3 = 0u;
                if(WIDE)
                {
                    p1 = half_of<T, true>(qw[WIDE][w]);
                    p3 = half_of<T, true>(qw[WIDE][w + 1]);
                    m1 = half_of<T, false>(qw[WIDE][w]);
                    m3 = half_of<T, false>(qw[WIDE][w + 1]);
                }
#pragma unroll
                for(int i = 0; i < NT; ++i)
                {
                    const uint4 lo = kb[i][0][j], hi = kb[i][1][j];
                    const uint32_t l0 = w ? lo.z : lo.x, l1 = w ? lo.w : lo.y;
                    const uint32_t h0 = w ? hi.z : hi.x, h1 = w ? hi.w : hi.y;
                    score_mma<T>(s[i], p0, p1, p2, p3, h0, h1);
                    score_mma<T>(s[i], m0, m1, m2, m3, l0, l1);
                    score_mma<T>(up[i], p0, p1, p2, p3, h0 & 0x7FFF7FFFu, h1 & 0x7FFF7FFFu);
                    score_mma<T>(down[i], m0, m1, m2, m3, l0 & 0x7FFF7FFFu, l1 & 0x7FFF7FFFu);
                }
            }
        }
#pragma unroll
        for(int i = 0; i < NT; ++i)
#pragma unroll
            for(int m = 0; m < (WIDE ? 2 : 1); ++m)
#pragma unroll
                for(int x = 0; x < 2; ++x)
                {
                    if(g0 + 8*m + n < a.group)
                    {
                        best[i][x] = max_nan(best[i][x], s[i][2*m + x]);
                        error[i][x] = max_nan(error[i][x], up[i][2*m + x] - down[i][2*m + x]);
                    }
                }
    }
#pragma unroll
    for(int i = 0; i < NT; ++i)
    {
#pragma unroll
        for(int x = 0; x < 2; ++x)
        {
#pragma unroll
            for(int o = 4; o < 32; o <<= 1)
            {
                best[i][x] = max_nan(best[i][x], __shfl_xor_sync(0xffffffffu, best[i][x], o));
                error[i][x] = max_nan(error[i][x], __shfl_xor_sync(0xffffffffu, error[i][x], o));
            }
            // column 2t + x of the tile is block 2t + x, whose bounds lane 4*(2t + x) loaded
            const bool gone = __shfl_sync(0xffffffffu, (int)missing[i], 4*(2*t + x)) != 0;
            const int block = block0 + 8*i + 2*t + x;
            if(n == 0 && block < count)
            {
                a.scores[(size_t)unit*a.max_blocks + block] = gone
                        ? make_float2(-CUDART_INF_F, 0.0f)
                        : make_float2(best[i][x], error[i][x]*SCORE_ERROR + SCORE_FLOOR);
            }
        }
    }
}

constexpr int PICK_THREADS = 512;
constexpr int PICK_WARPS = PICK_THREADS/32;
constexpr int PICK_LIST = 256;                   // near-ties that are ranked in shared memory

__device__ __forceinline__ int block_sum(int v, int *red)
{
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if((threadIdx.x & 31) == 0)
    {
        red[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    int all = 0;
#pragma unroll
    for(int w = 0; w < PICK_WARPS; ++w)
    {
        all += red[w];
    }
    return all;
}

// The num_selected best blocks of a unit, a CTA each.  CACHED: the scores are kept in
// shared memory (as many as the launch reserved), otherwise read from L2 again.
template<typename T, bool CACHED>
__global__ void __launch_bounds__(PICK_THREADS)
paged_pick_kernel(const PagedSelectArgs a)
{
    extern __shared__ float cached_s[];
    __shared__ int red[PICK_WARPS], red2[PICK_WARPS];
    __shared__ float fred[PICK_WARPS];
    __shared__ int listed_s, list_s[PICK_LIST];
    __shared__ unsigned long long list_key_s[PICK_LIST], cut_s;
    __shared__ int equal_want_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int unit = blockIdx.x, b = unit % a.batch, kvh = unit/a.batch;
    const int n = filled_blocks(a, b, nullptr), S = a.num_selected;
    int32_t *out = a.selected + (size_t)unit*S;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if(n <= S)
    {
        for(int i = tid; i < S; i += PICK_THREADS)
        {
            out[i] = i < n ? i : -1;
        }
        return;
    }
    const float2 *scores = a.scores + (size_t)unit*a.max_blocks;
    unsigned long long *keys = a.keys + (size_t)unit*a.max_blocks;
    // blocks that are always taken are out of the ranking
    const int begin = a.first_blocks, end = n - a.last_blocks;
    const int want = S - a.first_blocks - a.last_blocks;

    auto score = [&](int i) { return CACHED ? cached_s[i] : scores[i].x; };
    float error = 0.0f, low = CUDART_INF_F, high = -CUDART_INF_F;
    for(int i = begin + tid; i < end; i += PICK_THREADS)
    {
        const float2 se = scores[i];
        if(CACHED)
        {
            cached_s[i] = se.x;
        }
        error = max_nan(error, se.y);
        low = fminf(low, se.x);
        high = fmaxf(high, se.x);
    }
#pragma unroll
    for(int o = 16; o > 0; o >>= 1)
    {
        error = max_nan(error, __shfl_xor_sync(0xffffffffu, error, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    if(lane == 0)
    {
        fred[warp] = error;
        red[warp] = __float_as_int(low);
        red2[warp] = __float_as_int(high);
    }
    __syncthreads();
    for(int w = 0; w < PICK_WARPS; ++w)
    {
        error = max_nan(error, fred[w]);
        low = fminf(low, __int_as_float(red[w]));
        high = fmaxf(high, __int_as_float(red2[w]));
    }
    // no bound (NaN or infinite sums): every block is ranked exactly
    const bool unsure = !(error < CUDART_INF_F);
    float sure_in = CUDART_INF_F, sure_out = -CUDART_INF_F;
    if(want > 0 && !unsure)
    {
        // the want-th highest score: halve the range of keys; a threshold that exactly
        // `want` scores reach ends the search early
        uint32_t lo = score_key32(low), hi = score_key32(high);      // count(>= lo) >= want
        while(lo < hi)
        {
            const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;
            int c = 0;
            for(int i = begin + tid; i < end; i += PICK_THREADS)
            {
                c += score_key32(score(i)) >= mid ? 1 : 0;
            }
            c = block_sum(c, red);
            if(c >= want) lo = mid;
            else hi = mid - 1u;
            if(c == want)
            {
                break;
            }
        }
        // the least score that reaches it is the want-th highest
        float last = CUDART_INF_F;
        for(int i = begin + tid; i < end; i += PICK_THREADS)
        {
            const float s = score(i);
            last = score_key32(s) >= lo ? fminf(last, s) : last;
        }
#pragma unroll
        for(int o = 16; o > 0; o >>= 1)
        {
            last = fminf(last, __shfl_xor_sync(0xffffffffu, last, o));
        }
        __syncthreads();
        if(lane == 0)
        {
            fred[warp] = last;
        }
        __syncthreads();
        for(int w = 0; w < PICK_WARPS; ++w)
        {
            last = fminf(last, fred[w]);
        }
        // exact values are within `error` of the scores, the want-th of each as well; a few
        // units in the last place more cover these two sums
        const float band = last > -CUDART_INF_F ? 2.0f*error + fabsf(last)*4e-7f : 0.0f;
        sure_in = last + band;
        sure_out = last - band;
    }
    auto is_in = [&](float s) { return !unsure && s > sure_in; };
    auto is_near = [&](float s) { return unsure || (s <= sure_in && s >= sure_out); };
    bool take_near = false;                      // all near ones are taken; otherwise
    unsigned long long cut = 0ull;               // those above this key,
    int equal_want = 0;                          // and of those equal to it this many
    if(want > 0)
    {
        if(tid == 0)
        {
            listed_s = 0;
        }
        __syncthreads();
        int in = 0, near = 0;
        for(int i = begin + tid; i < end; i += PICK_THREADS)
        {
            const float s = score(i);
            in += is_in(s) ? 1 : 0;
            if(is_near(s))
            {
                ++near;
                const int at = atomicAdd(&listed_s, 1);
                if(at < PICK_LIST)
                {
                    list_s[at] = i;
                }
            }
        }
        in = block_sum(in, red);
        near = block_sum(near, red);
        const int need = want - in;              // of the near ones
        take_near = need >= near;
        if(!take_near)
        {
            const bool listed = near <= PICK_LIST;
            const int todo = listed ? near : end - begin;
            for(int k = warp; k < todo; k += PICK_WARPS)
            {
                const int i = listed ? list_s[k] : begin + k;
                if(!listed && !is_near(score(i)))
                {
                    continue;
                }
                const int page = a.block_table[(size_t)b*a.max_blocks + i];
                const unsigned long long key = page_in_pool(page, a.num_pages)
                        ? exact_key<T>(a, kvh, b, page, lane) : 0ull;
                if(lane == 0)
                {
                    keys[i] = key;
                    if(listed)
                    {
                        list_key_s[k] = key;
                    }
                }
            }
            __syncthreads();
            if(listed)
            {
                // the need-th highest key has fewer than need above it, need with its equals
                for(int k = tid; k < near; k += PICK_THREADS)
                {
                    const unsigned long long key = list_key_s[k];
                    int above = 0, equal = 0;
                    for(int j = 0; j < near; ++j)
                    {
                        above += list_key_s[j] > key ? 1 : 0;
                        equal += list_key_s[j] == key ? 1 : 0;
                    }
                    if(above < need && above + equal >= need)
                    {
                        cut_s = key;             // the same value from every equal
                        equal_want_s = need - above;
                    }
                }
                __syncthreads();
                cut = cut_s;
                equal_want = equal_want_s;
            }
            else
            {
                unsigned long long lo = 0ull, hi = ~0ull;
                while(lo < hi)
                {
                    const unsigned long long mid = lo + ((hi - lo) >> 1) + 1ull;
                    int c = 0;
                    for(int i = begin + tid; i < end; i += PICK_THREADS)
                    {
                        c += is_near(score(i)) && keys[i] >= mid ? 1 : 0;
                    }
                    c = block_sum(c, red);
                    if(c >= need) lo = mid;
                    else hi = mid - 1ull;
                }
                cut = lo;
                int above = 0;
                for(int i = begin + tid; i < end; i += PICK_THREADS)
                {
                    above += is_near(score(i)) && keys[i] > cut ? 1 : 0;
                }
                above = block_sum(above, red);
                equal_want = need - above;
            }
        }
        __syncthreads();
    }
    // write in index order: a run of neighbours a thread, one scan over the threads
    const int per = (n + PICK_THREADS - 1)/PICK_THREADS;
    const int i0 = min(n, tid*per), i1 = min(n, i0 + per);
    auto state = [&](int i)                      // 2 taken, 1 equal to the cut, 0 left out
    {
        if(i < begin || i >= end) return 2;
        if(want <= 0) return 0;
        const float s = score(i);
        if(is_in(s)) return 2;
        if(!is_near(s)) return 0;
        if(take_near) return 2;
        const unsigned long long key = keys[i];
        return key > cut ? 2 : key == cut ? 1 : 0;
    };
    int taken = 0, equal = 0;
    for(int i = i0; i < i1; ++i)
    {
        const int st = state(i);
        taken += st == 2 ? 1 : 0;
        equal += st == 1 ? 1 : 0;
    }
    int scan_t = taken, scan_e = equal;
#pragma unroll
    for(int o = 1; o < 32; o <<= 1)
    {
        const int ut = __shfl_up_sync(0xffffffffu, scan_t, o);
        const int ue = __shfl_up_sync(0xffffffffu, scan_e, o);
        scan_t += lane >= o ? ut : 0;
        scan_e += lane >= o ? ue : 0;
    }
    __syncthreads();
    if(lane == 31)
    {
        red[warp] = scan_t;
        red2[warp] = scan_e;
    }
    __syncthreads();
    int before_t = scan_t - taken, before_e = scan_e - equal;
    for(int w = 0; w < warp; ++w)
    {
        before_t += red[w];
        before_e += red2[w];
    }
    for(int i = i0; i < i1; ++i)
    {
        const int st = state(i);
        const bool take = st == 2 || (st == 1 && before_e < equal_want);
        const int at = before_t + min(before_e, equal_want);
        if(take && at < S)
        {
            out[at] = i;
        }
        before_t += st == 2 ? 1 : 0;
        before_e += st == 1 ? 1 : 0;
    }
}

static size_t select_bytes(int64_t units, int64_t max_blocks)
{
    return (size_t)units*max_blocks*(sizeof(float2) + sizeof(unsigned long long));
}

template<typename T, int DP, int NT>
static int launch_score(cudaStream_t s, const PagedSelectArgs &a)
{
    const int64_t per = SCORE_WARPS*8*NT;
    const int64_t ctas = (int64_t)a.batch*a.kv_heads*((a.max_blocks + per - 1)/per);
    if(ctas > INT32_MAX) return NNTILE_B200_E_SHAPE;
    if(a.group > 8) paged_score_kernel<T, DP, NT, true><<<(unsigned)ctas, SCORE_WARPS*32, 0, s>>>(a);
    else paged_score_kernel<T, DP, NT, false><<<(unsigned)ctas, SCORE_WARPS*32, 0, s>>>(a);
    return launch_status();
}

constexpr int PICK_CACHE_BYTES = 160 << 10;

template<typename T>
static int launch_pick(cudaStream_t s, const PagedSelectArgs &a)
{
    const bool cached = (int64_t)a.max_blocks*4 <= PICK_CACHE_BYTES;
    static PerDeviceOnce once;
    int dev = -1;
    if(cudaGetDevice(&dev) != cudaSuccess || !once.ensure(dev, []
    {
        return cudaFuncSetAttribute(paged_pick_kernel<T, true>,
                cudaFuncAttributeMaxDynamicSharedMemorySize, PICK_CACHE_BYTES) == cudaSuccess;
    }))
    {
        return NNTILE_B200_E_LAUNCH;
    }
    // starts while the scores are still being written and waits for them on the device
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = a.max_blocks > a.num_selected ? 1 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.batch*a.kv_heads);
    cfg.blockDim = dim3(PICK_THREADS);
    cfg.dynamicSmemBytes = cached ? (size_t)a.max_blocks*4 : 0;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t err = cached ? cudaLaunchKernelEx(&cfg, paged_pick_kernel<T, true>, a)
            : cudaLaunchKernelEx(&cfg, paged_pick_kernel<T, false>, a);
    if(err != cudaSuccess)
    {
        cudaGetLastError();
        return NNTILE_B200_E_LAUNCH;
    }
    return launch_status();
}

template<typename T>
static int select_impl(nntile_b200_stream_t stream, int64_t head, int64_t page_size,
        int64_t num_pages, int64_t max_blocks, int64_t batch, int64_t group, int64_t kv_heads,
        int64_t num_selected, int64_t first_blocks, int64_t last_blocks, const int32_t *lengths,
        const int32_t *block_table, const void *q, const void *bounds, int32_t *selected,
        void *workspace, size_t workspace_bytes, uint32_t *status)
{
    const int st = check_paged(head, page_size, num_pages, max_blocks, batch, kv_heads,
            NNTILE_B200_PAGES_SAME);
    if(st != NNTILE_B200_OK) return st;
    if(group < 0 || num_selected < 0 || first_blocks < 0 || last_blocks < 0) return NNTILE_B200_E_BADARG;
    if(num_selected > INT32_MAX || first_blocks > num_selected
            || last_blocks > num_selected - first_blocks)
    {
        return NNTILE_B200_E_BADARG;
    }
    if(group > 1 << 16 || batch*kv_heads*group > 1 << 24) return NNTILE_B200_E_SHAPE;
    if(batch == 0 || group == 0 || kv_heads == 0 || num_selected == 0) return NNTILE_B200_OK;
    if(!lengths || !q || !selected || !workspace || (max_blocks > 0 && !block_table)
            || (num_pages > 0 && !bounds))
    {
        return NNTILE_B200_E_BADARG;
    }
    if(((uintptr_t)q | (uintptr_t)bounds) & 1) return NNTILE_B200_E_ALIGN;
    if(((uintptr_t)lengths | (uintptr_t)block_table | (uintptr_t)selected | (uintptr_t)status) & 3)
    {
        return NNTILE_B200_E_ALIGN;
    }
    if(!aligned16(workspace)) return NNTILE_B200_E_ALIGN;
    const int64_t units = batch*kv_heads;
    if(workspace_bytes < select_bytes(units, max_blocks)) return NNTILE_B200_E_SCRATCH;
    PagedSelectArgs a;
    a.head = (int)head;
    a.page_size = (int)page_size;
    a.num_pages = (int)num_pages;
    a.max_blocks = (int)max_blocks;
    a.batch = (int)batch;
    a.group = (int)group;
    a.kv_heads = (int)kv_heads;
    a.num_selected = (int)num_selected;
    a.first_blocks = (int)first_blocks;
    a.last_blocks = (int)last_blocks;
    a.lengths = lengths;
    a.block_table = block_table;
    a.q = q;
    a.bounds = bounds;
    a.selected = selected;
    a.scores = static_cast<float2 *>(workspace);
    a.keys = reinterpret_cast<unsigned long long *>(a.scores + (size_t)units*max_blocks);
    a.status = status;
    const bool vec = head % 8 == 0 && aligned16(q) && aligned16(bounds);
    cudaStream_t s = as_stream(stream);
    int st2 = NNTILE_B200_OK;
    if(max_blocks > num_selected)                // otherwise everything is taken
    {
        if(vec && head <= 64) st2 = launch_score<T, 64, 4>(s, a);
        else if(vec && head <= 128) st2 = launch_score<T, 128, 2>(s, a);
        else if(vec) st2 = launch_score<T, 256, 1>(s, a);
        else
        {
            const int64_t ctas = units*((max_blocks + 3)/4);
            if(ctas > INT32_MAX) return NNTILE_B200_E_SHAPE;
            paged_score_generic_kernel<T><<<(unsigned)ctas, 128, 0, s>>>(a);
            st2 = launch_status();
        }
        if(st2 != NNTILE_B200_OK) return st2;
    }
    return launch_pick<T>(s, a);
}

} // namespace nb200

using namespace nb200;

extern "C" size_t nntile_b200_paged_select_workspace_bytes(int64_t max_blocks, int64_t batch,
        int64_t kv_heads)
{
    if(check_paged(1, 1, 0, max_blocks, batch, kv_heads, NNTILE_B200_PAGES_SAME)
            != NNTILE_B200_OK)
    {
        return 0;
    }
    return select_bytes(batch*kv_heads, max_blocks);
}

#define NB200_PAGED_SELECT_ENTRY(SFX, T) \
extern "C" int nntile_b200_paged_select_##SFX(nntile_b200_stream_t stream, int64_t head, \
        int64_t page_size, int64_t num_pages, int64_t max_blocks, int64_t batch, int64_t group, \
        int64_t kv_heads, int64_t num_selected, int64_t first_blocks, int64_t last_blocks, \
        const int32_t *lengths, const int32_t *block_table, const void *q, const void *bounds, \
        int32_t *selected, void *workspace, size_t workspace_bytes, uint32_t *status) \
{ \
    return select_impl<T>(stream, head, page_size, num_pages, max_blocks, batch, group, \
            kv_heads, num_selected, first_blocks, last_blocks, lengths, block_table, q, bounds, \
            selected, workspace, workspace_bytes, status); \
}

NB200_PAGED_SELECT_ENTRY(bf16, bf16)
NB200_PAGED_SELECT_ENTRY(fp16, __half)
