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
//
// Measured on one B200: 128 of up to 2049 blocks for 24 sequences and 8 kv heads of 128 (85.6 MB
// of bounds): 31-32 us, of which the scores are 20 and the ranking the rest, a chain of a
// dozen short passes; 64 of 4096 blocks of one sequence with the attention over them: 28 us, 30
// when the cache is not in L2.
// Scoring everything in 64 bits instead took 240 us for the first.
#include <algorithm>
#include <cfloat>

#include "paged.cuh"
#include "paged_rank.hh"
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

struct PagedSelectArgs
{
    int head, page_size, num_pages, max_blocks, batch, group, kv_heads, num_selected;
    int first_blocks, last_blocks;
    const int32_t *lengths, *block_table;
    const void *q, *bounds;
    int32_t *selected;
    float2 *scores;                              // [unit][block]: score, bound of its error
    unsigned long long *keys;                    // [unit][block]: exact, where it was needed
    bool vec;                                    // q and bounds allow 16-byte accesses
    uint32_t *status;
};

// One element's part of a score in 64 bits.  The product of two 16-bit factors is exact in 32
// bits while it is a normal number; the rest goes the long way, which also gives infinite and
// NaN bounds the value of the formula.
__device__ __forceinline__ double exact_term(float q, float low, float high)
{
    const float p = q*(q > 0.0f ? high : low), size = fabsf(p);
    const bool plain = size < 1e38f && (size > 1e-30f || q == 0.0f)
            && fabsf(low) < CUDART_INF_F && fabsf(high) < CUDART_INF_F;
    if(plain)
    {
        return (double)p;
    }
    return q != q ? (double)q : (double)fmaxf(q, 0.0f)*(double)high
            + (double)fminf(q, 0.0f)*(double)low;
}

// The exact key of a block for query head g, by 16 lanes (the same value in each of them;
// the whole warp takes part in the shuffles).
template<typename T>
__device__ __forceinline__ unsigned long long exact_key(const PagedSelectArgs &a, int kvh, int b,
        int page, int g)
{
    const int l16 = threadIdx.x & 15;
    const T *low = (const T *)a.bounds + ((size_t)page*a.kv_heads + kvh)*2*a.head;
    const T *high = low + a.head;
    const T *q = (const T *)a.q + (((size_t)kvh*a.group + g)*a.batch + b)*a.head;
    double s = 0.0;
    if(a.vec)
    {
        for(int h = 8*l16; h < a.head; h += 128)
        {
            const uint4 qv = *reinterpret_cast<const uint4 *>(q + h);
            const uint4 lv = *reinterpret_cast<const uint4 *>(low + h);
            const uint4 hv = *reinterpret_cast<const uint4 *>(high + h);
            const uint32_t qw[4] = {qv.x, qv.y, qv.z, qv.w};
            const uint32_t lw[4] = {lv.x, lv.y, lv.z, lv.w};
            const uint32_t hw[4] = {hv.x, hv.y, hv.z, hv.w};
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                const float2 x = unpack2<T>(qw[i]), y = unpack2<T>(lw[i]), z = unpack2<T>(hw[i]);
                s += exact_term(x.x, y.x, z.x) + exact_term(x.y, y.y, z.y);
            }
        }
    }
    else
    {
        for(int h = l16; h < a.head; h += 16)
        {
            s += exact_term(to_f(q[h]), to_f(low[h]), to_f(high[h]));
        }
    }
#pragma unroll
    for(int o = 8; o > 0; o >>= 1)
    {
        s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    return score_key(s);
}

__device__ __forceinline__ int filled_blocks(const PagedSelectArgs &a, int b, uint32_t *status)
{
    return blocks_of(checked_length(a.lengths, b, a.max_blocks*a.page_size, status), a.page_size);
}

// Any head: 16 lanes per block, sums in 64 bits, rounded once.
template<typename T>
__global__ void __launch_bounds__(128)
paged_score_generic_kernel(const PagedSelectArgs a)
{
    chain_wait();
    const int chunks = (a.max_blocks + 7)/8;
    const int unit = blockIdx.x/chunks;
    const int block = (blockIdx.x - unit*chunks)*8 + (threadIdx.x >> 4);
    const int b = unit % a.batch, kvh = unit/a.batch;
    const bool live = block < filled_blocks(a, b, a.status);
    const int page = live ? checked_page(a.block_table + (size_t)b*a.max_blocks, block,
            a.num_pages, a.status) : -1;
    unsigned long long key = 0ull;
    // without a pool there are no bounds to read, not even by lanes that only keep step
    for(int g = 0; g < (a.num_pages > 0 ? a.group : 0); ++g)
    {
        const unsigned long long one = exact_key<T>(a, kvh, b, max(page, 0), g);
        key = one > key ? one : key;
    }
    if(live && (threadIdx.x & 15) == 0)
    {
        float s = -CUDART_INF_F, error = 0.0f;
        if(page >= 0)
        {
            const double exact = __longlong_as_double((long long)((key >> 63)
                    ? key & 0x7FFFFFFFFFFFFFFFull : ~key));
            s = key == ~0ull ? CUDART_NAN_F : (float)exact;
            error = fabsf(s)*1.2e-7f + SCORE_FLOOR;      // infinite and NaN ones stay so
        }
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

// The positive and the negative parts of the two values of a word; NaN stays.
template<typename T> __device__ __forceinline__ uint32_t positive2(uint32_t w);
template<typename T> __device__ __forceinline__ uint32_t negative2(uint32_t w);
template<> __device__ __forceinline__ uint32_t positive2<bf16>(uint32_t w)
{
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
    return r;
}
template<> __device__ __forceinline__ uint32_t negative2<bf16>(uint32_t w)
{
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
    return r;
}
template<> __device__ __forceinline__ uint32_t positive2<__half>(uint32_t w)
{
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
    return r;
}
template<> __device__ __forceinline__ uint32_t negative2<__half>(uint32_t w)
{
    uint32_t r;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
    return r;
}

// Layout of the scoring kernel: a tile is 16 blocks of a unit, whose bounds (kmin, then kmax:
// 4*head contiguous bytes each) a warp copies into its private ring in shared memory and
// consumes itself; every warp of the grid takes the same number of neighbouring tiles.  The
// blocks are the 16 rows of the tensor instruction, 8 query heads its columns.  The order of
// the head elements is free in a sum, so a lane's 16-byte piece t + 4j of a row is the operand
// of two steps as it lies in memory.
constexpr int SCORE_WARPS = 8;
constexpr int SCORE_TILE = 16;
constexpr int SCORE_SMS = 148;

template<int DP>
struct ScoreTile
{
    static constexpr int HALF = DP/8;                    // 16-byte pieces of kmin, of kmax
    static constexpr int STAGE = SCORE_TILE*2*HALF*16;
    static constexpr int WARPS = DP == 256 ? 4 : SCORE_WARPS;
    static constexpr int RING = 196608/WARPS;
    static constexpr int STAGES = RING/STAGE < 8 ? RING/STAGE : 8;
    static constexpr int SMEM = WARPS*STAGES*STAGE;
    static constexpr int PASSES = SCORE_TILE*2*HALF/32;  // copies a lane issues a tile
    // the lanes that read together hold 4 pieces of 2 neighbouring rows: different banks
    static __device__ __forceinline__ int offset(int r, int c)
    {
        return r*2*HALF*16 + ((c ^ (((r & 1) << 2) | ((r >> 1) & 3))) << 4);
    }
};

// Tiles of a unit of sequence b, b's table held to its blocks.
__device__ __forceinline__ int score_tiles(const PagedSelectArgs &a, int b, uint32_t *status)
{
    const int blocks = filled_blocks(a, b, status);
    // otherwise all of them are taken
    return blocks > a.num_selected ? (blocks + SCORE_TILE - 1)/SCORE_TILE : 0;
}

template<typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(ScoreTile<DP>::WARPS*32, 1)
paged_score_kernel(const PagedSelectArgs a)
{
    using L = ScoreTile<DP>;
    constexpr int JN = DP/32, STAGES = L::STAGES, MT = WIDE ? 2 : 1;
    extern __shared__ __align__(128) uint8_t score_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = lane >> 2, t = lane & 3;
    uint8_t *ring = score_smem + warp*STAGES*L::STAGE;
    const int chunks = a.head/8;                          // of kmin
    for(int i = lane; a.head < DP && i < STAGES*L::STAGE/16; i += 32)
    {
        reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncwarp();
    chain_wait();

    // ---- this warp's share of all tiles, and the sequence it begins in
    int total = 0;
    for(int i0 = 0; i0 < a.batch; i0 += 32)
    {
        total += i0 + lane < a.batch ? score_tiles(a, i0 + lane,
                blockIdx.x == 0 && warp == 0 ? a.status : nullptr)*a.kv_heads : 0;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    const int workers = gridDim.x*L::WARPS, worker = blockIdx.x*L::WARPS + warp;
    const int share = (total + workers - 1)/workers;
    const int begin = (int)min((long long)total, (long long)worker*share);
    int left = min(share, total - begin);
    if(left <= 0)
    {
        return;
    }
    int b = 0, seq_begin = 0;
    for(int i0 = 0; i0 < a.batch; i0 += 32)
    {
        const int mine = i0 + lane < a.batch ? score_tiles(a, i0 + lane, nullptr)*a.kv_heads : 0;
        int scan = mine;
#pragma unroll
        for(int o = 1; o < 32; o <<= 1)
        {
            const int up = __shfl_up_sync(0xffffffffu, scan, o);
            scan += lane >= o ? up : 0;
        }
        const int all = __shfl_sync(0xffffffffu, scan, 31);
        if(seq_begin + all > begin)
        {
            const unsigned hit = __ballot_sync(0xffffffffu, seq_begin + scan > begin);
            const int k = __ffs((int)hit) - 1;
            b = i0 + k;
            seq_begin += __shfl_sync(0xffffffffu, scan - mine, k);
            break;
        }
        seq_begin += all;
    }

    // ---- issuing side
    int ib = b, ix = begin - seq_begin, ileft = left;
    int icount = filled_blocks(a, ib, nullptr), int_ = score_tiles(a, ib, nullptr);
    int ipos = 2;
    long long look_at = -1;
    auto issue = [&](int stage)
    {
        if(ileft > 0)
        {
            if(ix >= int_*a.kv_heads)
            {
                while(ix >= int_*a.kv_heads)
                {
                    ix -= int_*a.kv_heads;
                    ++ib;
                    int_ = score_tiles(a, ib, nullptr);
                }
                icount = filled_blocks(a, ib, nullptr);
                ipos = 2;
            }
            if(ipos == 2)
            {
                // bounds of the next 32 blocks: two tiles, which may be of two units
                ipos = 0;
                look_at = -1;
                const long long x = ix + (long long)(lane >> 4);
                if(x < (long long)int_*a.kv_heads && (lane >> 4) < ileft)
                {
                    const int kvh = (int)x/int_;
                    const int block = ((int)x - kvh*int_)*SCORE_TILE + (lane & 15);
                    if(block < icount)
                    {
                        const int page = checked_page(a.block_table + (size_t)ib*a.max_blocks,
                                block, a.num_pages, a.status);
                        look_at = page < 0 ? -1 : ((long long)page*a.kv_heads + kvh)*4*a.head;
                    }
                }
            }
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring + stage*L::STAGE);
#pragma unroll
            for(int i = 0; i < L::PASSES; ++i)
            {
                const int at = i*32 + lane, r = at/(2*L::HALF), c = at % (2*L::HALF);
                const long long from = __shfl_sync(0xffffffffu, look_at, 16*ipos + r);
                const int piece = c % L::HALF;
                if(from >= 0 && piece < chunks)
                {
                    const uint8_t *src = (const uint8_t *)a.bounds + from
                            + (piece + (c < L::HALF ? 0 : chunks))*16;
                    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;"
                            :: "r"(dst + L::offset(r, c)), "l"(src) : "memory");
                }
            }
            ++ipos;
            ++ix;
            --ileft;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for(int s = 0; s < STAGES - 1; ++s)
    {
        issue(s);
    }

    // ---- consuming side
    int nt = score_tiles(a, b, nullptr), count = filled_blocks(a, b, nullptr);
    int kvh = (begin - seq_begin)/nt, tile = (begin - seq_begin) - kvh*nt;
    bool fresh = true;
    uint32_t qp[MT][JN][4], qm[MT][JN][4];       // positive and negative parts of head 8m + n
    int stage = 0;
    while(left-- > 0)
    {
        asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 2) : "memory");
        __syncwarp();
        issue(stage == 0 ? STAGES - 1 : stage - 1);
        const uint8_t *st = ring + stage*L::STAGE;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        // of blocks n and n + 8, over this lane's heads
        float best[2] = {-CUDART_INF_F, -CUDART_INF_F}, error[2] = {0.0f, 0.0f};
        for(int g0 = 0; g0 < a.group; g0 += 8*MT)
        {
            if(fresh || a.group > 8*MT)
            {
#pragma unroll
                for(int m = 0; m < MT; ++m)
#pragma unroll
                    for(int j = 0; j < JN; ++j)
                    {
                        const int g = g0 + 8*m + n, h = 8*(t + 4*j);
                        const uint4 v = g < a.group && h < a.head
                                ? *reinterpret_cast<const uint4 *>((const T *)a.q
                                        + (((size_t)kvh*a.group + g)*a.batch + b)*a.head + h)
                                : make_uint4(0u, 0u, 0u, 0u);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for(int i = 0; i < 4; ++i)
                        {
                            qp[m][j][i] = positive2<T>(w[i]);
                            qm[m][j][i] = negative2<T>(w[i]);
                        }
                    }
                fresh = false;
            }
            // scores by the two parts of q (s, less) and their sums of magnitudes (up, down;
            // down is negative): four chains of products
            float s[MT][4] = {}, less[MT][4] = {}, up[MT][4] = {}, down[MT][4] = {};
#pragma unroll
            for(int j = 0; j < JN; ++j)
            {
                uint4 lo[2], hi[2];
#pragma unroll
                for(int x = 0; x < 2; ++x)
                {
                    lo[x] = *reinterpret_cast<const uint4 *>(st + L::offset(n + 8*x, t + 4*j));
                    hi[x] = *reinterpret_cast<const uint4 *>(st
                            + L::offset(n + 8*x, L::HALF + t + 4*j));
                }
#pragma unroll
                for(int w = 0; w < 4; w += 2)
                {
                    const uint32_t l0 = w ? lo[0].z : lo[0].x, l2 = w ? lo[0].w : lo[0].y;
                    const uint32_t l1 = w ? lo[1].z : lo[1].x, l3 = w ? lo[1].w : lo[1].y;
                    const uint32_t h0 = w ? hi[0].z : hi[0].x, h2 = w ? hi[0].w : hi[0].y;
                    const uint32_t h1 = w ? hi[1].z : hi[1].x, h3 = w ? hi[1].w : hi[1].y;
                    constexpr uint32_t ABS = 0x7FFF7FFFu;
#pragma unroll
                    for(int m = 0; m < MT; ++m)
                    {
                        score_mma<T>(s[m], h0, h1, h2, h3, qp[m][j][w], qp[m][j][w + 1]);
                        score_mma<T>(less[m], l0, l1, l2, l3, qm[m][j][w], qm[m][j][w + 1]);
                        score_mma<T>(up[m], h0 & ABS, h1 & ABS, h2 & ABS, h3 & ABS,
                                qp[m][j][w], qp[m][j][w + 1]);
                        score_mma<T>(down[m], l0 & ABS, l1 & ABS, l2 & ABS, l3 & ABS,
                                qm[m][j][w], qm[m][j][w + 1]);
                    }
                }
            }
            // value r: block n + 8*(r >> 1), head g0 + 8m + 2t + (r & 1)
#pragma unroll
            for(int m = 0; m < MT; ++m)
#pragma unroll
                for(int r = 0; r < 4; ++r)
                {
                    if(g0 + 8*m + 2*t + (r & 1) < a.group)
                    {
                        best[r >> 1] = max_nan(best[r >> 1], s[m][r] + less[m][r]);
                        error[r >> 1] = max_nan(error[r >> 1], up[m][r] - down[m][r]);
                    }
                }
        }
#pragma unroll
        for(int x = 0; x < 2; ++x)
        {
#pragma unroll
            for(int o = 1; o < 4; o <<= 1)
            {
                best[x] = max_nan(best[x], __shfl_xor_sync(0xffffffffu, best[x], o));
                error[x] = max_nan(error[x], __shfl_xor_sync(0xffffffffu, error[x], o));
            }
        }
        // lanes t = 0, 1 write blocks n and n + 8
        const int block = tile*SCORE_TILE + n + 8*t;
        if(t < 2 && block < count)
        {
            // the copying side has reported a missing page; its score is the lowest
            const bool gone = !page_in_pool(a.block_table[(size_t)b*a.max_blocks + block],
                    a.num_pages);
            a.scores[((size_t)kvh*a.batch + b)*a.max_blocks + block] = gone
                    ? make_float2(-CUDART_INF_F, 0.0f)
                    : make_float2(t ? best[1] : best[0],
                            (t ? error[1] : error[0])*SCORE_ERROR + SCORE_FLOOR);
        }
        if(++tile == nt)
        {
            tile = 0;
            fresh = true;
            if(++kvh == a.kv_heads && left > 0)
            {
                kvh = 0;
                do
                {
                    ++b;
                    nt = score_tiles(a, b, nullptr);
                }
                while(nt == 0);
                count = filled_blocks(a, b, nullptr);
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

// The bin, counted from the highest, in which the rank-th score lies: (bin, scores in it, rank
// inside it); by a warp, lane 31 - l having the eight from 8l on.
__device__ __forceinline__ void find_bin(const int *bins, int rank, int4 &found)
{
    const int lane = threadIdx.x & 31;
    const int4 c0 = *reinterpret_cast<const int4 *>(bins + 8*(31 - lane));
    const int4 c1 = *reinterpret_cast<const int4 *>(bins + 8*(31 - lane) + 4);
    const int c[8] = {c1.w, c1.z, c1.y, c1.x, c0.w, c0.z, c0.y, c0.x};
    const int sum = c[0] + c[1] + c[2] + c[3] + c[4] + c[5] + c[6] + c[7];
    int scan = sum;
#pragma unroll
    for(int o = 1; o < 32; o <<= 1)
    {
        const int up = __shfl_up_sync(0xffffffffu, scan, o);
        scan += lane >= o ? up : 0;
    }
    int above = scan - sum;
    if(above < rank && scan >= rank)
    {
#pragma unroll
        for(int k = 0; k < 8; ++k)
        {
            if(above < rank && above + c[k] >= rank)
            {
                found = make_int4(8*(31 - lane) + 7 - k, c[k], rank - above, 0);
            }
            above += c[k];
        }
    }
}

// Exact keys of listed blocks, the largest over the group; 16 lanes per block and query head,
// all threads of the block.  keys[] starts at zero, where a block without a page stays.
template<typename T, int THREADS>
__device__ void rank_near(const PagedSelectArgs &a, int kvh, int b, const int *list,
        unsigned long long *keys, int count)
{
    int c = (threadIdx.x >> 4)/a.group, g = (threadIdx.x >> 4) - c*a.group;
    const int dc = (THREADS/16)/a.group, dg = THREADS/16 - dc*a.group;
    while(__any_sync(0xffffffffu, c < count))
    {
        int page = -1;
        if(c < count)
        {
            page = a.block_table[(size_t)b*a.max_blocks + list[c]];
            page = page_in_pool(page, a.num_pages) ? page : -1;
        }
        if(__any_sync(0xffffffffu, page >= 0))
        {
            const unsigned long long key = exact_key<T>(a, kvh, b, max(page, 0), g);
            if(page >= 0 && (threadIdx.x & 15) == 0)
            {
                atomicMax(&keys[c], key);
            }
        }
        c += dc;
        g += dg;
        if(g >= a.group)
        {
            g -= a.group;
            ++c;
        }
    }
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
    __shared__ int listed_s, near_s, list_s[PICK_LIST];
    __shared__ unsigned long long list_key_s[PICK_LIST], cut_s;
    __shared__ int equal_want_s;
    __shared__ __align__(16) int bin_s[256];
    __shared__ int4 hit_s;
    __shared__ float list_score_s[PICK_LIST], last_s;
    __shared__ uint2 mask_s[PICK_THREADS];
    __shared__ int2 before_s[PICK_THREADS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int unit = blockIdx.x, b = unit % a.batch, kvh = unit/a.batch;
    // behind the scoring kernel the lengths are settled; as the first kernel of a call (a table
    // that short is taken whole) this one has to wait for them
    const bool scored = a.max_blocks > a.num_selected;
    if(!scored)
    {
        chain_wait();
    }
    const int n = filled_blocks(a, b, a.status), S = a.num_selected;
    int32_t *out = a.selected + (size_t)unit*S;
    if(scored)
    {
        chain_wait();
    }
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
    // eight at a time: the first pass is one latency of the L2 cache for up to 4096 blocks
    for(int i0 = begin + tid; i0 < end; i0 += 8*PICK_THREADS)
    {
        float2 se[8];
#pragma unroll
        for(int u = 0; u < 8; ++u)
        {
            const int i = i0 + u*PICK_THREADS;
            se[u] = i < end ? scores[i] : make_float2(0.0f, -1.0f);
        }
#pragma unroll
        for(int u = 0; u < 8; ++u)
        {
            const int i = i0 + u*PICK_THREADS;
            if(i < end)
            {
                if(CACHED)
                {
                    cached_s[i] = se[u].x;
                }
                error = max_nan(error, se[u].y);
                low = fminf(low, se[u].x);
                high = fmaxf(high, se[u].x);
            }
        }
    }
#pragma unroll
    for(int o = 16; o > 0; o >>= 1)
    {
        error = max_nan(error, __shfl_xor_sync(0xffffffffu, error, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    for(int i = tid; i < 256; i += PICK_THREADS)
    {
        bin_s[i] = 0;
    }
    if(tid == 0)
    {
        listed_s = 0;
    }
    if(lane == 0)
    {
        fred[warp] = error;
        red[warp] = __float_as_int(low);
        red2[warp] = __float_as_int(high);
    }
    __syncthreads();
#pragma unroll
    for(int w = 0; w < PICK_WARPS; ++w)
    {
        error = max_nan(error, fred[w]);
        low = fminf(low, __int_as_float(red[w]));
        high = fmaxf(high, __int_as_float(red2[w]));
    }
    // no bound (NaN or infinite sums): every block is ranked exactly
    const bool unsure = !(error < CUDART_INF_F);
    float sure_in = CUDART_INF_F, sure_out = -CUDART_INF_F;
    // The usual case in few passes: 256 equal bins of the range; the want-th score lies in one
    // of them, and what may be exchanged with it in that one and its neighbours, a hundred
    // blocks or so.  They are ranked in shared memory, the near-ties among them exactly, and
    // the outcome replaces their scores.
    bool decided = false;
    if(CACHED && want > 0 && !unsure && low < high && low > -FLT_MAX)
    {
        const float origin = 0.5f*low, scale = 256.0f/(0.5f*high - origin);
        auto bin = [&](float s) { return min(255, (int)((0.5f*s - origin)*scale)); };
#pragma unroll 4
        for(int i = begin + tid; i < end; i += PICK_THREADS)
        {
            atomicAdd(&bin_s[bin(cached_s[i])], 1);
        }
        __syncthreads();
        if(warp == 0)
        {
            find_bin(bin_s, want, hit_s);
        }
        __syncthreads();
        const int hit = hit_s.x, above = want - hit_s.z;         // scores in higher bins
        const int over = hit < 255 ? bin_s[hit + 1] : 0;
        const int many = hit_s.y + over + (hit > 0 ? bin_s[hit - 1] : 0);
        const float widest = 2.0f*error + fmaxf(fabsf(low), fabsf(high))*4e-7f;
        // the neighbours hold all that is near: half of the band's width is in the scale
        decided = many <= PICK_LIST && 0.5f*widest*scale < 0.9f;
        if(decided)
        {
#pragma unroll 4
            for(int i = begin + tid; i < end; i += PICK_THREADS)
            {
                const float s = cached_s[i];
                const int d = bin(s) - hit;
                if(d >= -1 && d <= 1)
                {
                    const int at = atomicAdd(&listed_s, 1);
                    list_s[at] = i;
                    list_score_s[at] = s;
                }
            }
            __syncthreads();
            // PICK_LIST <= PICK_THREADS: an entry a thread
            const int rank = want - above + over;                // among the listed ones
            const float mine = tid < many ? list_score_s[tid] : 0.0f;
            int higher = 0, same = 0;
            for(int j = 0; tid < many && j < many; ++j)
            {
                higher += list_score_s[j] > mine ? 1 : 0;
                same += list_score_s[j] == mine ? 1 : 0;
            }
            if(tid < many && higher < rank && higher + same >= rank)
            {
                last_s = mine;                                   // the same from every equal
            }
            if(tid == 0)
            {
                near_s = 0;
            }
            __syncthreads();
            const float last = last_s, band = 2.0f*error + fabsf(last)*4e-7f;
            sure_in = last + band;
            const bool near = tid < many && mine <= sure_in && mine >= last - band;
            int slot = 0;
            if(near)
            {
                slot = atomicAdd(&near_s, 1);
            }
            const int block = tid < many ? list_s[tid] : 0;
            // what is above the band in the list is taken; the rest of `rank` are near ones
            const int need = rank - __syncthreads_count(tid < many && mine > sure_in);
            const int nears = near_s;
            if(near)
            {
                list_s[slot] = block;
                list_key_s[slot] = 0ull;
                // all of them, unless they are ranked
                cached_s[block] = CUDART_INF_F;
            }
            __syncthreads();
            if(need < nears)
            {
                rank_near<T, PICK_THREADS>(a, kvh, b, list_s, list_key_s, nears);
                __syncthreads();
                for(int k = tid; k < nears; k += PICK_THREADS)
                {
                    const unsigned long long key = list_key_s[k];
                    int better = 0;
                    for(int j = 0; j < nears; ++j)
                    {
                        better += list_key_s[j] > key || (list_key_s[j] == key
                                && list_s[j] < list_s[k]) ? 1 : 0;
                    }
                    if(better >= need)
                    {
                        cached_s[list_s[k]] = -CUDART_INF_F;
                    }
                }
            }
            __syncthreads();
        }
        else
        {
            __syncthreads();
            for(int i = tid; i < 256; i += PICK_THREADS)
            {
                bin_s[i] = 0;
            }
            __syncthreads();
        }
    }
    if(want > 0 && !unsure && !decided)
    {
        // The want-th highest score: count the scores in up to 256 equal bins of the range of
        // their keys; the bin it lies in holds a few, which are ranked against one another - or,
        // when they are more than the list, is the range of another round.  On keys and not on
        // the scores, so that every round divides the range, whatever the scores are.  Missing
        // pages (-inf) go into the lowest bin.
        int rank = want;                         // from the top of the range
        auto key = [&](int i) { return score_key32(fmaxf(score(i), -FLT_MAX)); };
        RankRange range = rank_range(score_key32(fmaxf(low, -FLT_MAX)),
                score_key32(fmaxf(high, -FLT_MAX)));
        while(range.low < range.high)
        {
#pragma unroll 4
            for(int i = begin + tid; i < end; i += PICK_THREADS)
            {
                const uint32_t k = key(i);
                if(rank_inside(range, k))
                {
                    atomicAdd(&bin_s[rank_bin(range, k)], 1);
                }
            }
            __syncthreads();
            if(warp == 0)
            {
                find_bin(bin_s, rank, hit_s);
            }
            __syncthreads();
            const int hits = hit_s.y;
            rank = hit_s.z;
            range = rank_narrowed(range, hit_s.x);
            if(hits <= PICK_LIST && range.low < range.high)
            {
#pragma unroll 4
                for(int i = begin + tid; i < end; i += PICK_THREADS)
                {
                    const uint32_t k = key(i);
                    if(rank_inside(range, k))
                    {
                        list_score_s[atomicAdd(&listed_s, 1)] = score_of_key(k);
                    }
                }
                __syncthreads();
                for(int k = tid; k < hits; k += PICK_THREADS)
                {
                    const float s = list_score_s[k];
                    int over = 0, same = 0;
                    for(int j = 0; j < hits; ++j)
                    {
                        over += list_score_s[j] > s ? 1 : 0;
                        same += list_score_s[j] == s ? 1 : 0;
                    }
                    if(over < rank && over + same >= rank)
                    {
                        last_s = s;              // the same value from every equal
                    }
                }
                __syncthreads();
                range.low = range.high = score_key32(last_s);
                break;
            }
            for(int i = tid; i < 256; i += PICK_THREADS)
            {
                bin_s[i] = 0;
            }
            __syncthreads();
        }
        const float lowest = score_of_key(range.low);
        const float last = lowest > -FLT_MAX ? lowest : -CUDART_INF_F;
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
    if(want > 0 && !decided)
    {
        if(tid == 0)
        {
            listed_s = 0;
        }
        __syncthreads();
        int in = 0, near = 0;
#pragma unroll 4
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
                    list_key_s[at] = 0ull;
                }
            }
        }
        in = __reduce_add_sync(0xffffffffu, in);
        if(lane == 0)
        {
            red[warp] = in;
        }
        __syncthreads();
        near = listed_s;
        in = 0;
#pragma unroll
        for(int w = 0; w < PICK_WARPS; ++w)
        {
            in += red[w];
        }
        const int need = want - in;              // of the near ones
        take_near = need >= near;
        if(!take_near)
        {
            const bool listed = near <= PICK_LIST;
            if(listed)
            {
                rank_near<T, PICK_THREADS>(a, kvh, b, list_s, list_key_s, near);
            }
            else
            {
                // More than the list holds: rows of NaN and infinities, a query of zeros, blocks
                // whose bounds are all alike.  Every block is summed again, near or not.
                for(int i0 = begin; i0 < end; i0 += PICK_LIST)
                {
                    const int count = min(PICK_LIST, end - i0);
                    __syncthreads();
                    for(int k = tid; k < count; k += PICK_THREADS)
                    {
                        list_s[k] = i0 + k;
                        list_key_s[k] = 0ull;
                    }
                    __syncthreads();
                    rank_near<T, PICK_THREADS>(a, kvh, b, list_s, list_key_s, count);
                    __syncthreads();
                    for(int k = tid; k < count; k += PICK_THREADS)
                    {
                        keys[i0 + k] = list_key_s[k];
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
                for(int k = tid; k < near; k += PICK_THREADS)
                {
                    keys[list_s[k]] = list_key_s[k];
                }
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
    auto state = [&](int i)                      // 2 taken, 1 equal to the cut, 0 left out
    {
        if(i < begin || i >= end) return 2;
        if(want <= 0) return 0;
        const float s = score(i);
        if(is_in(s)) return 2;
        if(decided || !is_near(s)) return 0;
        if(take_near) return 2;
        const unsigned long long key = keys[i];
        return key > cut ? 2 : key == cut ? 1 : 0;
    };
    // write in index order: 32 neighbours a warp as two masks, a thread per mask for the sums
    int taken = 0, equals = 0;                   // of the runs before
    for(int base = 0; base < n; base += 32*PICK_THREADS)
    {
        __syncthreads();
#pragma unroll 2
        for(int k = warp; k < PICK_THREADS && base + 32*k < n; k += PICK_WARPS)
        {
            const int i = base + 32*k + lane;
            const int st = i < n ? state(i) : 0;
            const unsigned take = __ballot_sync(0xffffffffu, st == 2);
            const unsigned equal = __ballot_sync(0xffffffffu, st == 1);
            if(lane == 0)
            {
                mask_s[k] = make_uint2(take, equal);
            }
        }
        __syncthreads();
        uint2 mine = make_uint2(0u, 0u);
        if(base + 32*tid < n)
        {
            mine = mask_s[tid];
        }
        const int ct = __popc(mine.x), ce = __popc(mine.y);
        int scan_t = ct, scan_e = ce;
#pragma unroll
        for(int o = 1; o < 32; o <<= 1)
        {
            const int ut = __shfl_up_sync(0xffffffffu, scan_t, o);
            const int ue = __shfl_up_sync(0xffffffffu, scan_e, o);
            scan_t += lane >= o ? ut : 0;
            scan_e += lane >= o ? ue : 0;
        }
        if(lane == 31)
        {
            red[warp] = scan_t;
            red2[warp] = scan_e;
        }
        __syncthreads();
        int before_t = taken + scan_t - ct, before_e = equals + scan_e - ce;
#pragma unroll
        for(int w = 0; w < PICK_WARPS; ++w)
        {
            before_t += w < warp ? red[w] : 0;
            before_e += w < warp ? red2[w] : 0;
            taken += red[w];
            equals += red2[w];
        }
        before_s[tid] = make_int2(before_t, before_e);
        __syncthreads();
        for(int k = warp; k < PICK_THREADS && base + 32*k < n; k += PICK_WARPS)
        {
            const uint2 mask = mask_s[k];
            const int2 before = before_s[k];
            const unsigned below = (1u << lane) - 1u;
            const bool equal = (mask.y >> lane & 1u) != 0u;
            const int e = before.y + __popc(mask.y & below);
            const int at = before.x + __popc(mask.x & below) + min(e, equal_want);
            if((((mask.x >> lane & 1u) != 0u) || (equal && e < equal_want)) && at < S)
            {
                out[at] = base + 32*k + lane;
            }
        }
    }
}

// Blocks of a table and of a selection: loops of the kernels here step past their ends, in 32
// bits.
constexpr int64_t SELECT_MOST = (int64_t)1 << 30;

static size_t select_bytes(int64_t units, int64_t max_blocks)
{
    return (size_t)units*max_blocks*(sizeof(float2) + sizeof(unsigned long long));
}

template<typename T, int DP, bool WIDE>
static int launch_score_as(cudaStream_t s, const PagedSelectArgs &a, unsigned grid)
{
    static PerDeviceOnce once;
    int dev = -1;
    if(cudaGetDevice(&dev) != cudaSuccess || !once.ensure(dev, []
    {
        return cudaFuncSetAttribute(paged_score_kernel<T, DP, WIDE>,
                cudaFuncAttributeMaxDynamicSharedMemorySize, ScoreTile<DP>::SMEM) == cudaSuccess;
    }))
    {
        return NNTILE_B200_E_LAUNCH;
    }
    return launch_chained(paged_score_kernel<T, DP, WIDE>, dim3(grid), ScoreTile<DP>::WARPS*32,
            ScoreTile<DP>::SMEM, s, a);
}

template<typename T, int DP>
static int launch_score(cudaStream_t s, const PagedSelectArgs &a)
{
    constexpr int WARPS = ScoreTile<DP>::WARPS;
    const int64_t tiles = (int64_t)a.batch*a.kv_heads
            *((a.max_blocks + SCORE_TILE - 1)/SCORE_TILE);
    const unsigned grid = (unsigned)std::min<int64_t>(SCORE_SMS, (tiles + WARPS - 1)/WARPS);
    return a.group > 8 ? launch_score_as<T, DP, true>(s, a, grid)
            : launch_score_as<T, DP, false>(s, a, grid);
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
    // set up while the scores are still being written, and waits for them on the device
    const dim3 grid((unsigned)a.batch*a.kv_heads);
    return cached ? launch_chained(paged_pick_kernel<T, true>, grid, PICK_THREADS,
                    (size_t)a.max_blocks*4, s, a)
            : launch_chained(paged_pick_kernel<T, false>, grid, PICK_THREADS, 0, s, a);
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
    if(group > 1 << 16 || batch*kv_heads*group > 1 << 24 || max_blocks > SELECT_MOST
            || num_selected > SELECT_MOST)
    {
        return NNTILE_B200_E_SHAPE;
    }
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
    // 16-byte rows; for the tensor instruction also tiles that 30 bits can count
    a.vec = head % 8 == 0 && aligned16(q) && aligned16(bounds);
    const bool vec = a.vec && units*((max_blocks + SCORE_TILE - 1)/SCORE_TILE) < (int64_t)1 << 30;
    cudaStream_t s = as_stream(stream);
    int st2 = NNTILE_B200_OK;
    if(max_blocks > num_selected)                // otherwise everything is taken
    {
        if(vec && head <= 64) st2 = launch_score<T, 64>(s, a);
        else if(vec && head <= 128) st2 = launch_score<T, 128>(s, a);
        else if(vec) st2 = launch_score<T, 256>(s, a);
        else
        {
            const int64_t ctas = units*((max_blocks + 7)/8);
            if(ctas > INT32_MAX) return NNTILE_B200_E_SHAPE;
            st2 = launch_chained(paged_score_generic_kernel<T>, dim3((unsigned)ctas), 128, 0, s,
                    a);
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
            != NNTILE_B200_OK || max_blocks > SELECT_MOST)
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
