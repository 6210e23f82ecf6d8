// Attention of one new token per sequence over a paged key/value cache.
//
// o = sum_i p_i v_i / sum_i p_i,  p_i = exp(q.k_i/sqrt(head)), over the filled positions of
// a sequence, or over those of them that lie in the blocks a list selects.
#include <algorithm>

#include "paged.cuh"

namespace nb200 {

constexpr int PD_WARPS = 4;
constexpr float PD_LOG2E = 1.4426950408889634f;
constexpr float PD_LN2 = 0.6931471805599453f;

struct PagedDecodeArgs
{
    int head, page_size, num_pages, max_blocks, batch, group, kv_heads, num_selected;
    float scale_log2;                    // log2(e)/sqrt(head)
    const int32_t *lengths, *block_table, *selected;
    const void *q, *k_pages, *v_pages;
    const uint8_t *k_scales, *v_scales;
    void *out;
    float *lse_out;
    float *part_o, *part_lse;
    uint32_t *status;
    int nsplit, chunk;                   // chunk: list positions per split (blocks)
};

// Any head up to 256, any page size, any alignment: a warp takes a position at a time,
// CUDA-core dot products, the cache re-read once per query head of a group.
template<typename T, bool E4M3, int EPL>
__global__ void __launch_bounds__(PD_WARPS*32)
paged_decode_generic_kernel(const PagedDecodeArgs a)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int split = blockIdx.x % a.nsplit;
    const int qh = blockIdx.x/a.nsplit;                  // (kvh*group + g)*batch + b
    const int b = qh % a.batch, kvh = qh/(a.batch*a.group);
    const int D = a.head;
    const int len = checked_length(a.lengths, b, a.max_blocks*a.page_size, a.status);
    const int blocks = blocks_of(len, a.page_size);
    const int listed = a.selected ? a.num_selected : blocks;
    const int32_t *list = a.selected
            ? a.selected + ((size_t)kvh*a.batch + b)*a.num_selected : nullptr;
    const int32_t *table = a.block_table + (size_t)b*a.max_blocks;
    const T *q = (const T *)a.q + (size_t)qh*D;
    float qv[EPL], o[EPL];
#pragma unroll
    for(int x = 0; x < EPL; ++x)
    {
        const int h = lane + 32*x;
        qv[x] = h < D ? to_f(q[h])*a.scale_log2 : 0.0f;
        o[x] = 0.0f;
    }
    float top = -CUDART_INF_F, sum = 0.0f;
    const int j_end = min(listed, (split + 1)*a.chunk);
    for(int j = split*a.chunk; j < j_end; ++j)
    {
        int block = j;
        if(list)
        {
            bool bad = false;
            block = held_block(list[j], blocks, a.max_blocks, bad);
            if(bad)
            {
                report(a.status, NNTILE_B200_PAGED_BAD_BLOCK);
            }
            if(block < 0)
            {
                continue;
            }
        }
        const int page = checked_page(table, block, a.num_pages, a.status);
        if(page < 0)
        {
            continue;
        }
        const int rows = min(a.page_size, len - block*a.page_size);
        const size_t row0 = ((size_t)page*a.kv_heads + kvh)*a.page_size;
        for(int r = warp; r < rows; r += PD_WARPS)
        {
            const size_t at = (row0 + r)*D;
            float part = 0.0f, ks = 1.0f, vs = 1.0f;
            if(E4M3)
            {
                ks = scale_value(a.k_scales[row0 + r]);
                vs = scale_value(a.v_scales[row0 + r]);
            }
#pragma unroll
            for(int x = 0; x < EPL; ++x)
            {
                const int h = lane + 32*x;
                float kv = 0.0f;
                if(h < D)
                {
                    kv = E4M3 ? e4m3x2_to_f2(((const uint8_t *)a.k_pages)[at + h]).x
                            : to_f(((const T *)a.k_pages)[at + h]);
                }
                part = fmaf(qv[x], kv, part);
            }
            const float s = warp_sum(part)*ks;
            const float ntop = fmaxf(top, s);
            // every score so far -inf: nothing to weigh yet (and no inf - inf below)
            const float shrink = top == ntop ? 1.0f : exp2f(top - ntop);
            const float p = s == -CUDART_INF_F ? 0.0f : exp2f(s - ntop);
            sum = sum*shrink + p;
            top = ntop;
#pragma unroll
            for(int x = 0; x < EPL; ++x)
            {
                const int h = lane + 32*x;
                float vv = 0.0f;
                if(h < D)
                {
                    vv = E4M3 ? e4m3x2_to_f2(((const uint8_t *)a.v_pages)[at + h]).x*vs
                            : to_f(((const T *)a.v_pages)[at + h]);
                }
                o[x] = fmaf(p, vv, o[x]*shrink);
            }
        }
    }
    __shared__ float o_s[PD_WARPS][PAGED_MAX_HEAD];
    __shared__ float top_s[PD_WARPS], sum_s[PD_WARPS];
    if(lane == 0)
    {
        top_s[warp] = top;
        sum_s[warp] = sum;
    }
#pragma unroll
    for(int x = 0; x < EPL; ++x)
    {
        const int h = lane + 32*x;
        if(h < D)
        {
            o_s[warp][h] = o[x];
        }
    }
    __syncthreads();
    float big = -CUDART_INF_F;
    for(int w = 0; w < PD_WARPS; ++w)
    {
        big = fmaxf(big, top_s[w]);
    }
    for(int d = threadIdx.x; d < D; d += PD_WARPS*32)
    {
        float den = 0.0f, num = 0.0f;
        for(int w = 0; w < PD_WARPS; ++w)
        {
            if(sum_s[w] != 0.0f)
            {
                const float wgt = exp2f(top_s[w] - big);
                den += wgt*sum_s[w];
                num += wgt*o_s[w][d];
            }
        }
        const size_t slot = (size_t)qh*a.nsplit + split;
        a.part_o[slot*D + d] = den != 0.0f ? num/den : 0.0f;
        if(d == 0)
        {
            a.part_lse[slot] = den != 0.0f ? big + log2f(den) : -CUDART_INF_F;
        }
    }
}

// Joins the splits of a query head by log-sum-exp weights; a warp per head.
template<typename T>
__global__ void __launch_bounds__(128)
paged_decode_join_kernel(const PagedDecodeArgs a, int heads)
{
    const int lane = threadIdx.x & 31;
    const int qh = blockIdx.x*4 + (threadIdx.x >> 5);
    if(qh >= heads)
    {
        return;
    }
    const float *lse = a.part_lse + (size_t)qh*a.nsplit;
    float big = -CUDART_INF_F;
    for(int s = lane; s < a.nsplit; s += 32)
    {
        big = max_nan(big, lse[s]);
    }
#pragma unroll
    for(int o = 16; o > 0; o >>= 1)
    {
        big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, o));
    }
    const bool empty = big == -CUDART_INF_F;
    float den = 0.0f;
    for(int s = lane; s < a.nsplit; s += 32)
    {
        den += empty ? 0.0f : exp2f(lse[s] - big);
    }
    den = warp_sum(den);
    for(int d = lane; d < a.head; d += 32)
    {
        float num = 0.0f;
        for(int s = 0; s < a.nsplit; ++s)
        {
            const float l = lse[s];
            if(l != -CUDART_INF_F)
            {
                num += exp2f(l - big)*a.part_o[((size_t)qh*a.nsplit + s)*a.head + d];
            }
        }
        ((T *)a.out)[(size_t)qh*a.head + d] = from_f<T>(empty ? 0.0f : num/den);
    }
    if(lane == 0 && a.lse_out)
    {
        a.lse_out[qh] = empty ? -CUDART_INF_F : (big + log2f(den))*PD_LN2;
    }
}

struct PagedDecodePlan
{
    int nsplit, chunk;
    size_t bytes;
};

static PagedDecodePlan paged_decode_plan(int64_t head, int64_t page_size, int64_t max_blocks,
        int64_t batch, int64_t group, int64_t kv_heads, int64_t num_selected)
{
    PagedDecodePlan p;
    const int64_t listed = num_selected > 0 ? num_selected : max_blocks;
    const int64_t heads = batch*group*kv_heads;
    int64_t nsplit = (148*8 + heads - 1)/std::max<int64_t>(heads, 1);
    const int64_t rows = listed*page_size;
    nsplit = std::min(nsplit, (rows + 255)/256);
    nsplit = std::max<int64_t>(1, std::min(nsplit, std::max<int64_t>(listed, 1)));
    const int64_t chunk = std::max<int64_t>(1, (listed + nsplit - 1)/nsplit);
    p.chunk = (int)chunk;
    p.nsplit = (int)std::max<int64_t>(1, (listed + chunk - 1)/chunk);
    p.bytes = (size_t)heads*p.nsplit*(size_t)(head + 1)*sizeof(float);
    return p;
}

template<typename T>
static int decode_impl(nntile_b200_stream_t stream, int64_t head, int64_t page_size,
        int64_t num_pages, int64_t max_blocks, int64_t batch, int64_t group, int64_t kv_heads,
        int64_t num_selected, int page_format, const int32_t *lengths,
        const int32_t *block_table, const int32_t *selected, const void *q, const void *k_pages,
        const void *v_pages, const uint8_t *k_scales, const uint8_t *v_scales, void *out,
        float *lse_out, void *workspace, size_t workspace_bytes, uint32_t *status)
{
    const int st = check_paged(head, page_size, num_pages, max_blocks, batch, kv_heads,
            page_format);
    if(st != NNTILE_B200_OK) return st;
    if(group < 0 || num_selected < 0) return NNTILE_B200_E_BADARG;
    if(num_selected > INT32_MAX/page_size || group > 1 << 16 || batch*kv_heads*group > 1 << 24)
    {
        return NNTILE_B200_E_SHAPE;
    }
    if(batch == 0 || group == 0 || kv_heads == 0) return NNTILE_B200_OK;
    const bool e4m3 = page_format == NNTILE_B200_PAGES_E4M3;
    if(!lengths || !q || !out || !workspace || (max_blocks > 0 && !block_table)
            || (num_selected > 0 && !selected) || (num_pages > 0 && (!k_pages || !v_pages
            || (e4m3 && (!k_scales || !v_scales)))))
    {
        return NNTILE_B200_E_BADARG;
    }
    if(((uintptr_t)q | (uintptr_t)out) & 1) return NNTILE_B200_E_ALIGN;
    if(!e4m3 && (((uintptr_t)k_pages | (uintptr_t)v_pages) & 1)) return NNTILE_B200_E_ALIGN;
    if(((uintptr_t)lengths | (uintptr_t)block_table | (uintptr_t)selected | (uintptr_t)lse_out
            | (uintptr_t)status) & 3)
    {
        return NNTILE_B200_E_ALIGN;
    }
    if(!aligned16(workspace)) return NNTILE_B200_E_ALIGN;
    const PagedDecodePlan plan = paged_decode_plan(head, page_size, max_blocks, batch, group,
            kv_heads, num_selected);
    if(workspace_bytes < plan.bytes) return NNTILE_B200_E_SCRATCH;
    const int64_t heads = batch*group*kv_heads;
    if(heads*plan.nsplit > INT32_MAX) return NNTILE_B200_E_SHAPE;
    PagedDecodeArgs a;
    a.head = (int)head;
    a.page_size = (int)page_size;
    a.num_pages = (int)num_pages;
    a.max_blocks = (int)max_blocks;
    a.batch = (int)batch;
    a.group = (int)group;
    a.kv_heads = (int)kv_heads;
    a.num_selected = (int)num_selected;
    a.scale_log2 = PD_LOG2E/sqrtf((float)head);
    a.lengths = lengths;
    a.block_table = block_table;
    a.selected = num_selected > 0 ? selected : nullptr;
    a.q = q;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    a.out = out;
    a.lse_out = lse_out;
    a.part_o = static_cast<float *>(workspace);
    a.part_lse = a.part_o + (size_t)heads*plan.nsplit*(size_t)head;
    a.status = status;
    a.nsplit = plan.nsplit;
    a.chunk = plan.chunk;
    cudaStream_t s = as_stream(stream);
    const unsigned grid = (unsigned)(heads*plan.nsplit);
    const int epl = (int)((head + 31)/32);
#define NB200_PD(E, N) paged_decode_generic_kernel<T, E, N><<<grid, PD_WARPS*32, 0, s>>>(a)
#define NB200_PD_N(E) \
    do { \
        if(epl <= 1) NB200_PD(E, 1); \
        else if(epl <= 2) NB200_PD(E, 2); \
        else if(epl <= 4) NB200_PD(E, 4); \
        else NB200_PD(E, 8); \
    } while(0)
    if(e4m3) NB200_PD_N(true);
    else NB200_PD_N(false);
#undef NB200_PD_N
#undef NB200_PD
    if(launch_status() != NNTILE_B200_OK) return NNTILE_B200_E_LAUNCH;
    paged_decode_join_kernel<T><<<(unsigned)((heads + 3)/4), 128, 0, s>>>(a, (int)heads);
    return launch_status();
}

} // namespace nb200

using namespace nb200;

extern "C" size_t nntile_b200_paged_decode_sdpa_workspace_bytes(int64_t head, int64_t page_size,
        int64_t max_blocks, int64_t batch, int64_t group, int64_t kv_heads, int64_t num_selected)
{
    if(check_paged(head, page_size, 0, max_blocks, batch, kv_heads, NNTILE_B200_PAGES_SAME)
            != NNTILE_B200_OK || group < 0 || group > 1 << 16 || num_selected < 0
            || num_selected > INT32_MAX/page_size)
    {
        return 0;
    }
    return paged_decode_plan(head, page_size, max_blocks, batch, group, kv_heads,
            num_selected).bytes;
}

#define NB200_PAGED_DECODE_ENTRY(SFX, T) \
extern "C" int nntile_b200_paged_decode_sdpa_##SFX(nntile_b200_stream_t stream, int64_t head, \
        int64_t page_size, int64_t num_pages, int64_t max_blocks, int64_t batch, int64_t group, \
        int64_t kv_heads, int64_t num_selected, int page_format, const int32_t *lengths, \
        const int32_t *block_table, const int32_t *selected, const void *q, \
        const void *k_pages, const void *v_pages, const uint8_t *k_scales, \
        const uint8_t *v_scales, void *out, float *lse_out, void *workspace, \
        size_t workspace_bytes, uint32_t *status) \
{ \
    return decode_impl<T>(stream, head, page_size, num_pages, max_blocks, batch, group, \
            kv_heads, num_selected, page_format, lengths, block_table, selected, q, k_pages, \
            v_pages, k_scales, v_scales, out, lse_out, workspace, workspace_bytes, status); \
}

NB200_PAGED_DECODE_ENTRY(bf16, bf16)
NB200_PAGED_DECODE_ENTRY(fp16, __half)
