// Shared pieces of the paged key/value cache kernels (paged_cache.cu,
// paged_decode.cu, paged_select.cu).
//
// A cache is a pool of pages; a page holds `page_size` consecutive positions of one
// sequence for every kv head, and a (page, kv head) pair is one contiguous row-major
// [page_size][head] block.  block_table[b][n] names the page that holds positions
// n*page_size .. of sequence b.  Lengths and tables live in device memory, so every
// kernel checks what it reads there: a page outside the pool, a length outside the table
// or a selected block outside the table is left out and reported in the caller's
// status word, never dereferenced.
//
// 8-bit pages hold e4m3 codes and one exponent byte per (position, kv head) row: a value
// is code * 2^(byte - 127).  The scale is a power of two on purpose: dividing by it and
// multiplying by it are exact, so a stored row has one possible value (no dependence on
// how a reciprocal rounds), every stored value is a bf16 number, and a kernel may fold
// the scale into its scores without a rounding of its own.  e4m3 is a floating format, so
// a power of two costs no relative precision against an arbitrary scale, only up to one
// binade at the small end of its range.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged_check.hh"

namespace nb200 {

constexpr int PAGED_MAX_HEAD = 256;

__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template<typename T> __device__ __forceinline__ T from_f(float x);
template<> __device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16_rn(x); }
template<> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// the two values of a 32-bit word, low half first, and back
template<typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template<> __device__ __forceinline__ float2 unpack2<bf16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template<> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w)
{
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}
template<typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template<> __device__ __forceinline__ uint32_t pack2<bf16>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template<> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// the same, cut off towards zero instead of rounded
template<typename T> __device__ __forceinline__ uint32_t cut2(float lo, float hi);
template<> __device__ __forceinline__ uint32_t cut2<bf16>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template<> __device__ __forceinline__ uint32_t cut2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// the larger and the smaller of two pairs; a NaN loses
template<typename T> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
template<> __device__ __forceinline__ uint32_t max2<bf16>(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template<> __device__ __forceinline__ uint32_t max2<__half>(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template<typename T> __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b);
template<> __device__ __forceinline__ uint32_t min2<bf16>(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template<> __device__ __forceinline__ uint32_t min2<__half>(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// two e4m3 codes (low byte first) -> two halves; exact, every e4m3 value is an fp16 value
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two_codes)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two_codes));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t two_codes)
{
    return unpack2<__half>(e4m3x2_to_half2(two_codes));
}
// round to nearest even; the caller keeps finite values within +-448
__device__ __forceinline__ uint32_t f2_to_e4m3x2(float lo, float hi)
{
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// 2^(byte - 127)
__device__ __forceinline__ float scale_value(uint32_t byte)
{
    return byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
// Exponent byte of a row whose largest finite magnitude is `amax`: the smallest e with
// amax * 2^-e <= 448 = 1.75 * 2^8, so compare the fraction bits with those of 1.75.
__device__ __forceinline__ uint32_t scale_byte(float amax)
{
    const uint32_t bits = __float_as_uint(amax);
    if(bits == 0u)
    {
        return 127u;
    }
    const int byte = (int)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (uint32_t)(byte < 1 ? 1 : byte);
}
// 2^-(byte - 127), byte in [1, 247] as scale_byte returns
__device__ __forceinline__ float inverse_scale(uint32_t byte)
{
    return __uint_as_float((254u - byte) << 23);
}

__device__ __forceinline__ float min_nan(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void report(uint32_t *status, uint32_t bit)
{
    if(status)
    {
        atomicOr(status, bit);
    }
}

// Filled positions of sequence b, held inside what its table can name.
__device__ __forceinline__ int checked_length(const int32_t *lengths, int b, int capacity,
        uint32_t *status)
{
    bool bad = false;
    const int len = held_length(lengths[b], capacity, bad);
    if(bad)
    {
        report(status, NNTILE_B200_PAGED_BAD_LENGTH);
    }
    return len;
}

// Page that holds block n of a sequence, or -1 when the table names none in the pool.
__device__ __forceinline__ int checked_page(const int32_t *table, int n, int num_pages,
        uint32_t *status)
{
    const int page = table[n];
    if(!page_in_pool(page, num_pages))
    {
        report(status, NNTILE_B200_PAGED_BAD_PAGE);
        return -1;
    }
    return page;
}

// Chained launches.  A kernel of this family may be set up while the one before it in the
// stream still runs; it touches memory only after chain_wait(), which returns when everything
// before it is complete and visible, and only then lets the next one be set up.  So whatever
// starts early starts after all but the last kernel before it are complete: what that one
// does not write (for the second kernel of a call: lengths and tables) may be read before the
// wait, the rest only after it.  Every kernel waits, also in blocks with nothing to do: a
// grid must not end before the one it is chained to.  What it reads may still be written while
// it is being set up, so no pointer of a chained kernel is promised to be read-only
// (`const __restrict__`, __ldg): such loads could be moved ahead of the wait.
__device__ __forceinline__ void chain_wait()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template<typename... P, typename... A>
inline int launch_chained(void (*kernel)(P...), dim3 grid, int threads, size_t smem,
        cudaStream_t s, A... args)
{
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...) != cudaSuccess)
    {
        cudaGetLastError();
        return NNTILE_B200_E_LAUNCH;
    }
    return launch_status();
}

// Sizes every paged entry point shares.  max_blocks*page_size positions are addressed
// with 32-bit integers; byte offsets into the pool are 64-bit everywhere.
inline int check_paged(int64_t head, int64_t page_size, int64_t num_pages, int64_t max_blocks,
        int64_t batch, int64_t kv_heads, int page_format)
{
    if(head < 1 || page_size < 1 || num_pages < 0 || max_blocks < 0 || batch < 0 || kv_heads < 0
            || (page_format != NNTILE_B200_PAGES_SAME && page_format != NNTILE_B200_PAGES_E4M3))
    {
        return NNTILE_B200_E_BADARG;
    }
    const int64_t lim = INT32_MAX;
    if(head > PAGED_MAX_HEAD || page_size > 65536 || num_pages > lim || max_blocks > lim/page_size
            || batch > 1 << 20 || kv_heads > 1 << 16 || batch*kv_heads > 1 << 24)
    {
        return NNTILE_B200_E_SHAPE;
    }
    return NNTILE_B200_OK;
}

} // namespace nb200
