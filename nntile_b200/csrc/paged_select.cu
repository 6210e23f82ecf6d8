// Choosing the blocks of a paged cache that a new token attends to.
//
// For query heads q_g (g < group) and the bounds kmin, kmax of a block's stored keys,
//     score = max_g sum_d max(q_gd, 0)*kmax_d + min(q_gd, 0)*kmin_d,
// the least upper bound on q_g.k over every key inside the bounds.  The blocks with the
// highest scores are selected, ties by the lowest index, so the answer is a set that does
// not depend on the order of any sum: scores are compared as 64-bit sums of exact
// products.
#include <algorithm>

#include "paged.cuh"

namespace nb200 {

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

// keys[unit][block], a warp per block.
template<typename T>
__global__ void __launch_bounds__(128)
paged_score_kernel(int head, int page_size, int num_pages, int max_blocks, int batch, int group,
        int kv_heads, const int32_t *__restrict__ lengths,
        const int32_t *__restrict__ block_table, const T *__restrict__ q,
        const T *__restrict__ bounds, unsigned long long *__restrict__ keys,
        uint32_t *__restrict__ status)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = (max_blocks + 3)/4;
    const int unit = blockIdx.x/chunks;
    const int block = (blockIdx.x - unit*chunks)*4 + warp;
    const int b = unit % batch, kvh = unit/batch;
    const int len = checked_length(lengths, b, max_blocks*page_size, status);
    if(block >= max_blocks || (int64_t)block*page_size >= len)
    {
        return;
    }
    const int page = checked_page(block_table + (size_t)b*max_blocks, block, num_pages, status);
    unsigned long long best = 0ull;
    if(page >= 0)
    {
        const T *low = bounds + ((size_t)page*kv_heads + kvh)*2*head, *high = low + head;
        for(int g = 0; g < group; ++g)
        {
            const T *qg = q + ((size_t)(kvh*group + g)*batch + b)*head;
            double s = 0.0;
            for(int h = lane; h < head; h += 32)
            {
                const double x = (double)to_f(qg[h]);
                s += (x > 0.0 ? x : 0.0)*(double)to_f(high[h])
                        + (x < 0.0 ? x : 0.0)*(double)to_f(low[h]);
            }
#pragma unroll
            for(int o = 16; o > 0; o >>= 1)
            {
                s += __shfl_xor_sync(0xffffffffu, s, o);
            }
            const unsigned long long key = score_key(s);
            best = key > best ? key : best;
        }
    }
    if(lane == 0)
    {
        keys[(size_t)unit*max_blocks + block] = best;
    }
}

constexpr int PICK_THREADS = 256;

// The num_selected highest keys of a unit: radix selection, eight bits a pass from the
// top, for the value of the last key that is taken; then one pass in index order writes
// what is above it and as many of its equals as are still wanted.
__global__ void __launch_bounds__(PICK_THREADS)
paged_pick_kernel(int page_size, int max_blocks, int batch, int num_selected, int first_blocks,
        int last_blocks, const int32_t *__restrict__ lengths,
        const unsigned long long *__restrict__ keys, int32_t *__restrict__ selected)
{
    const int unit = blockIdx.x, b = unit % batch;
    const int n = blocks_of(checked_length(lengths, b, max_blocks*page_size, nullptr), page_size);
    const unsigned long long *key = keys + (size_t)unit*max_blocks;
    int32_t *out = selected + (size_t)unit*num_selected;
    const int tid = threadIdx.x;
    if(n <= num_selected)
    {
        for(int i = tid; i < num_selected; i += PICK_THREADS)
        {
            out[i] = i < n ? i : -1;
        }
        return;
    }
    __shared__ unsigned hist[256];
    __shared__ unsigned long long prefix_s;
    __shared__ int want_s;
    __shared__ int above_s[PICK_THREADS/32], equal_s[PICK_THREADS/32];
    // a block that is always taken is out of the ranking
    const int free_end = n - last_blocks;
    int want = num_selected - first_blocks - last_blocks;
    unsigned long long prefix = 0ull, mask = 0ull;
    if(want > 0)
    {
        for(int shift = 56; shift >= 0; shift -= 8)
        {
            for(int i = tid; i < 256; i += PICK_THREADS)
            {
                hist[i] = 0u;
            }
            __syncthreads();
            for(int i = first_blocks + tid; i < free_end; i += PICK_THREADS)
            {
                if((key[i] & mask) == prefix)
                {
                    atomicAdd(&hist[(unsigned)(key[i] >> shift) & 255u], 1u);
                }
            }
            __syncthreads();
            if(tid == 0)
            {
                int left = want, d = 255;
                while(d > 0 && (int)hist[d] < left)
                {
                    left -= (int)hist[d--];
                }
                want_s = left;
                prefix_s = prefix | (unsigned long long)d << shift;
            }
            __syncthreads();
            want = want_s;
            prefix = prefix_s;
            mask |= 255ull << shift;
            __syncthreads();
        }
    }
    // `want` equals of `prefix` are taken, the lowest indices first
    int taken = 0, equals = 0;
    for(int i0 = 0; i0 < n; i0 += PICK_THREADS)
    {
        const int i = i0 + tid;
        const bool forced = i < n && (i < first_blocks || i >= free_end);
        const bool ranked = i < n && !forced && num_selected > first_blocks + last_blocks;
        const bool above = forced || (ranked && key[i] > prefix);
        const bool equal = ranked && key[i] == prefix;
        const unsigned ma = __ballot_sync(0xffffffffu, above);
        const unsigned me = __ballot_sync(0xffffffffu, equal);
        const int lane = tid & 31, warp = tid >> 5;
        if(lane == 0)
        {
            above_s[warp] = __popc(ma);
            equal_s[warp] = __popc(me);
        }
        __syncthreads();
        int a = 0, e = 0, all_a = 0, all_e = 0;
        for(int w = 0; w < PICK_THREADS/32; ++w)
        {
            a += w < warp ? above_s[w] : 0;
            e += w < warp ? equal_s[w] : 0;
            all_a += above_s[w];
            all_e += equal_s[w];
        }
        const unsigned before = (1u << lane) - 1u;
        const int ea = equals + e + __popc(me & before);            // equals before this one
        const int at = taken + a + __popc(ma & before) + min(ea, want)
                - min(equals, want);
        if((above || (equal && ea < want)) && at < num_selected)
        {
            out[at] = i;
        }
        taken += all_a + min(equals + all_e, want) - min(equals, want);
        equals += all_e;
        __syncthreads();
    }
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
    if(workspace_bytes < (size_t)units*max_blocks*sizeof(unsigned long long))
    {
        return NNTILE_B200_E_SCRATCH;
    }
    cudaStream_t s = as_stream(stream);
    const int64_t ctas = units*((max_blocks + 3)/4);
    if(ctas > INT32_MAX) return NNTILE_B200_E_SHAPE;
    unsigned long long *keys = static_cast<unsigned long long *>(workspace);
    if(ctas > 0)
    {
        paged_score_kernel<T><<<(unsigned)ctas, 128, 0, s>>>((int)head, (int)page_size,
                (int)num_pages, (int)max_blocks, (int)batch, (int)group, (int)kv_heads, lengths,
                block_table, (const T *)q, (const T *)bounds, keys, status);
        if(launch_status() != NNTILE_B200_OK) return NNTILE_B200_E_LAUNCH;
    }
    paged_pick_kernel<<<(unsigned)units, PICK_THREADS, 0, s>>>((int)page_size, (int)max_blocks,
            (int)batch, (int)num_selected, (int)first_blocks, (int)last_blocks, lengths, keys,
            selected);
    return launch_status();
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
    return (size_t)batch*kv_heads*max_blocks*sizeof(unsigned long long);
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
