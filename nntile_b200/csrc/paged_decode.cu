// Attention of one new token per sequence over a paged key/value cache.
//
// o = sum_i p_i v_i / sum_i p_i,  p_i = exp(q.k_i/sqrt(head)), over the filled positions of
// a sequence, or over those of them that lie in the blocks a list selects.
//
// Every key and value is used for 2*group multiply-adds per byte or less: the kernel is
// bound by HBM bandwidth when the cache is long and by latency when it is short, so the
// design is about bytes in flight and about even shares:
//   - work is cut into tiles of 16 positions.  All tiles of all (sequence, kv head) units
//     stand in one row, and every worker takes the same number of neighbours, whatever
//     the lengths are (they are only known on the device), or, where few units allow it, an
//     even piece of one unit.  A unit that falls into several shares is joined by a second,
//     small kernel;
//   - a warp copies its own tiles into a private ring in shared memory (cp.async, 16 bytes a
//     lane, swizzled; rows behind the length are zero-filled, never read) and is its own
//     consumer: no barrier inside a share.  24 KB a warp, 192 KB an SM, more than four times
//     what HBM latency times bandwidth asks for; the ring runs on across units;
//   - page numbers are looked up 32 tiles at a time, a lane each, ahead of the ring;
//   - scores and weighted values go through the warp-level tensor instruction (m16n8k16, fp32
//     accumulate), transposed: keys and columns of V are its 16 rows, 8 query heads its
//     columns, so no row is idle for groups up to 8 and the accumulators take half the
//     registers of the other way round.  The weights go in twice (fp16) or three times (bf16),
//     in 16 bits and what these lose, and so count with 22 or 24 bits;
//   - weights refer to an exponent that follows the maximum only when a score passes it by
//     2^4: most tiles need one vote instead of a maximum over lanes and a pass over the
//     accumulators;
//   - 8-bit rows are widened to fp16, exactly, on their way into the operands; their scales go
//     into scores and weights, where they are powers of two;
//   - sums are fp32 and round to nearest: a tile's products leave the tensor instruction, which
//     cuts off, before they are added to the others, and sums of weights are compensated.
//
// Measured on one B200 (copy bandwidth 6 553 GB/s), head 128: 64 sequences of 8192, 8 kv heads,
// group 4, bf16: 332-338 us, 6.4 TB/s; 37 sequences of up to 16383, e4m3, group 8: 138-158 us,
// 4.9-5.6 TB/s; one of 100003, 2 kv heads, group 7, fp16: 25 us, 4.1 TB/s, of which 15.6 us are
// the bytes and the rest the start (length, page and first row, one after the other), the
// slowest SM and the joining (18-19 us where the cache, 102 MB, is in L2 from the call before).
// With 8-bit heads of 64 the instructions bound it (300 MB in 75 us), with 16-bit rows the copies
// do.  The choices below were measured with inputs that together exceed L2, unless they say
// otherwise.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "per_device.hh"

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
    float2 *part_sums;
    int2 *spans;                         // [unit]: first and last worker that has a part of it
    uint32_t *status;
    int wpw;                             // warps of a worker
    int whole;                           // workers take whole units, nothing is joined
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
    // sums of RUN positions, and of what was summed before: like terms, thousands of them in a
    // row, would all round the same way
    constexpr int RUN = 64;
    float qv[EPL], o[EPL], run_o[EPL];
#pragma unroll
    for(int x = 0; x < EPL; ++x)
    {
        const int h = lane + 32*x;
        qv[x] = h < D ? to_f(q[h])*a.scale_log2 : 0.0f;
        o[x] = run_o[x] = 0.0f;
    }
    float top = -CUDART_INF_F, sum = 0.0f, run_sum = 0.0f;
    int run = 0;
    auto end_run = [&]()
    {
        sum += run_sum;
        run_sum = 0.0f;
        run = 0;
#pragma unroll
        for(int x = 0; x < EPL; ++x)
        {
            o[x] += run_o[x];
            run_o[x] = 0.0f;
        }
    };
    const int j_end = split_end(listed, split, a.chunk);
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
            const float p = s == -CUDART_INF_F ? 0.0f : exp2f(s - ntop);
            if(top != ntop)
            {
                const float shrink = exp2f(top - ntop);
                end_run();
                sum *= shrink;
#pragma unroll
                for(int x = 0; x < EPL; ++x)
                {
                    o[x] *= shrink;
                }
                top = ntop;
            }
            run_sum += p;
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
                run_o[x] = fmaf(p, vv, run_o[x]);
            }
            if(++run == RUN)
            {
                end_run();
            }
        }
    }
    end_run();
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

// ------------------------------------------------------------------ tensor-core kernel

constexpr int PD_SMS = 148;
constexpr int PD_TILE = 16;                  // positions of a tile
// Sequences up to which a warp adds up their tiles by itself: against the block's prefix sums
// 25.6 us and 26.5 for one of 100003, 15.1 and 17.2 for 33 of 2000, 90.7 and 91.6 for 64 of 2000
// with 8 kv heads.
constexpr int PD_BATCH = 64;

// Warps of a block, one block per SM: with four, 16-bit rows of 256 columns still have three
// tiles (48 KB) a warp in the ring; their 8-bit rows are bound by instructions and take eight
// (59 us for 300 MB against 72 with four).
__host__ __device__ constexpr int paged_warps(bool e4m3, int dp)
{
    return dp == 256 && !e4m3 ? 4 : 8;
}

// Layout of one kernel variant.  DP: head size rounded up to 64, 128 or 256 (columns behind
// the head stay zero in the ring); MT: tiles of 8 query heads that share a pass.
template<bool E4M3, int DP>
struct PagedTile
{
    static constexpr int WARPS = paged_warps(E4M3, DP);
    static constexpr int ROW_BYTES = DP*(E4M3 ? 1 : 2);
    static constexpr int CHUNKS = ROW_BYTES/16;          // 16-byte pieces of a row
    static constexpr int KV_BYTES = PD_TILE*ROW_BYTES;   // one of K, V
    static constexpr int STAGE = 2*KV_BYTES + (E4M3 ? 2*PD_TILE : 0);
    static constexpr int RING = 198144/WARPS;
    static constexpr int STAGES = RING/STAGE < 12 ? RING/STAGE : 12;
    // Tiles a warp takes at once.  A tile is one chain (scores, weights, values) of several
    // hundred cycles; short rows put two or four side by side, so that 8 warps ask for bytes
    // as fast as HBM delivers them (8-bit heads of 64 with four 75 us for 300 MB, with two 82;
    // 8-bit heads of 128 with two 61, with one 65; 16-bit heads of 64 with two 55, with one 56).
    static constexpr int ABREAST = 8192/(2*KV_BYTES) < 1 ? 1 : 8192/(2*KV_BYTES);
    static constexpr int AHEAD = STAGES - ABREAST;       // tiles in flight or waiting
    static_assert(AHEAD >= ABREAST, "the ring must hold what is consumed and what is coming");
    static constexpr int MBLK = DP/16;                   // 16-column blocks of the output
    // One tile of 8 heads of every warp, for 256 columns in two rounds: with 16-bit rows of
    // 256 that leaves an SM room for blocks of the joining kernel, which then wait beside this
    // one (16 kv heads of 512 positions 12.1 -> 11.3 us).  With 128 columns the second round
    // costs as much as it gains.
    static constexpr int ROUNDS = DP == 256 ? 2 : 1;
    static constexpr int MERGE = WARPS*8*DP*4/ROUNDS;
    static constexpr int SMEM = WARPS*STAGES*STAGE + MERGE;

    // Offset of piece c of row r.  A 128-byte line holds 8 pieces; which of them is piece c
    // depends on the row, so that the lanes that load together hit different banks: 8 rows,
    // one piece (ldmatrix, 16-bit rows); 2 neighbouring rows, 4 pieces (8-bit keys: `rot`
    // puts the row's last bit on top); 4 even rows, 2 pieces (8-bit values).
    static __device__ __forceinline__ int offset(int r, int c, bool rot)
    {
        if(ROW_BYTES == 64)      // two rows a line
        {
            return (r >> 1)*128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
        }
        const int x = rot ? ((r & 1) << 2) | ((r >> 1) & 3) : r & 7;
        return r*ROW_BYTES + ((c ^ x) << 4);
    }
    // Column of the output that row n (x = 0) or n + 8 (x = 1) of accumulator block i holds.
    static __device__ __forceinline__ int column(int i, int x, int n)
    {
        if(!E4M3) return 16*i + 8*x + n;
        return DP == 64 ? 8*n + 2*i + x : (i >> 3)*128 + 16*n + 2*(i & 7) + x;
    }
};

__device__ __forceinline__ uint32_t smem_addr(const void *p)
{
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" :: "r"(dst), "l"(src),
            "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template<int N>
__device__ __forceinline__ void copy_wait()
{
    asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// T: the operand format, bf16 or __half
template<typename T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
        uint32_t a3, uint32_t b0, uint32_t b1);
template<>
__device__ __forceinline__ void mma16<bf16>(float (&c)[4], uint32_t a0, uint32_t a1,
        uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template<>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], uint32_t a0, uint32_t a1,
        uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a + b and a - b of two values an instruction
__device__ __forceinline__ void plus2(float (&r)[2], const float (&a)[2], const float (&b)[2])
{
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
            "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
            : "=f"(r[0]), "=f"(r[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
}
__device__ __forceinline__ void minus2(float (&r)[2], const float (&a)[2], const float (&b)[2])
{
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
            "sub.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
            : "=f"(r[0]), "=f"(r[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
}
// c += o, two values an instruction
__device__ __forceinline__ void add4(float (&c)[4], const float (&o)[4])
{
#pragma unroll
    for(int i = 0; i < 4; i += 2)
    {
        asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
                "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
                : "+f"(c[i]), "+f"(c[i + 1]) : "f"(o[i]), "f"(o[i + 1]));
    }
}
// transposes an 8x8 matrix of 16-bit values held as an accumulator's words
__device__ __forceinline__ uint32_t transpose8x8(uint32_t w)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ float ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t word4(const uint4 &v, int i)
{
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Tiles of one unit of sequence b.
__device__ __forceinline__ int unit_tiles(const PagedDecodeArgs &a, int len)
{
    if(a.selected)
    {
        return len > 0 ? a.num_selected*(a.page_size/PD_TILE) : 0;
    }
    return (len + PD_TILE - 1)/PD_TILE;
}

// Exclusive prefix sums of the tiles of the sequences, prefix[0..batch]; all threads of the
// block, a barrier at the end.
__device__ __forceinline__ void tile_prefix(const PagedDecodeArgs &a, int units_per_seq,
        int *prefix, int *warp_sums, bool reporting)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthreads = blockDim.x;
    const int per = (a.batch + nthreads - 1)/nthreads;
    const int b0 = min(a.batch, tid*per), b1 = min(a.batch, b0 + per);
    int sum = 0;
    for(int b = b0; b < b1; ++b)
    {
        const int len = checked_length(a.lengths, b, a.max_blocks*a.page_size,
                reporting ? a.status : nullptr);
        sum += unit_tiles(a, len)*units_per_seq;
        prefix[b + 1] = sum;
    }
    int scan = sum;
#pragma unroll
    for(int o = 1; o < 32; o <<= 1)
    {
        const int up = __shfl_up_sync(0xffffffffu, scan, o);
        scan += lane >= o ? up : 0;
    }
    if(lane == 31)
    {
        warp_sums[warp] = scan;
    }
    __syncthreads();
    int before = scan - sum;
    for(int w = 0; w < warp; ++w)
    {
        before += warp_sums[w];
    }
    for(int b = b0; b < b1; ++b)
    {
        prefix[b + 1] += before;
    }
    if(tid == 0)
    {
        prefix[0] = 0;
    }
    __syncthreads();
}

__device__ __forceinline__ int held_len(const PagedDecodeArgs &a, int b)
{
    bool bad = false;
    return held_length(a.lengths[b], a.max_blocks*a.page_size, bad);
}

// The four values of accumulator block i (columns n and n + 8 of it, heads 8m + 2t and
// 8m + 2t + 1), either final or into part `part` of the workspace: [part][m][head][column].
template<typename T, bool E4M3, int DP, int MT>
__device__ __forceinline__ void write_part(const PagedDecodeArgs &a, bool complete, int part,
        int m, int lane, int i, const float (&z)[4], const float (&den)[2], int kvh, int h0,
        int heads, int b)
{
    using L = PagedTile<E4M3, DP>;
    const int n = lane >> 2, t = lane & 3;
#pragma unroll
    for(int y = 0; y < 2; ++y)
    {
        const int g = 8*m + 2*t + y;
        if(g >= heads)
        {
            continue;
        }
        if(!complete)
        {
            float *o = a.part_o + (((size_t)part*MT + m)*8 + 2*t + y)*DP;
            o[L::column(i, 0, n)] = z[y];
            o[L::column(i, 1, n)] = z[2 + y];
        }
        else
        {
            const float inv = den[y] == 0.0f ? 0.0f : 1.0f/den[y];
            T *out = (T *)a.out + (((size_t)kvh*a.group + h0 + g)*a.batch + b)*a.head;
            const int c0 = L::column(i, 0, n), c1 = L::column(i, 1, n);
            if(c0 < a.head)
            {
                out[c0] = from_f<T>(z[y]*inv);
            }
            if(c1 < a.head)
            {
                out[c1] = from_f<T>(z[2 + y]*inv);
            }
        }
    }
}

// Reference exponent and sum of head `head` of tile m.
template<int MT>
__device__ __forceinline__ void write_sums(const PagedDecodeArgs &a, bool complete, int part,
        int m, int head, float top, float sum, int kvh, int h0, int heads, int b)
{
    const int g = 8*m + head;
    if(g >= heads)
    {
        return;
    }
    if(!complete)
    {
        a.part_sums[((size_t)part*MT + m)*8 + head] = make_float2(top, sum);
    }
    else if(a.lse_out)
    {
        a.lse_out[((size_t)kvh*a.group + h0 + g)*a.batch + b] = sum == 0.0f ? -CUDART_INF_F
                : ((top == -CUDART_INF_F ? 0.0f : top) + log2f(sum))*PD_LN2;
    }
}

// How the tiles are dealt out: `workers` shares of `share` neighbouring tiles, a worker
// being a warp (wpw = 1) or a block (wpw = its warps).
struct PagedShares
{
    int wpw, workers, share;
};

template<int WARPS>
__host__ __device__ inline PagedShares paged_shares(int total, int blocks, int wpw)
{
    PagedShares s;
    s.wpw = wpw;
    s.workers = blocks*(WARPS/s.wpw);
    s.share = (total + s.workers - 1)/s.workers;
    s.share = (s.share + s.wpw - 1)/s.wpw*s.wpw;
    return s;
}

// ceil(tiles/size), 0 <= tiles < 2^30, the quotient below 2^20: exact, and shorter than the
// division of integers that the start of a call would otherwise wait for several times.
__device__ __forceinline__ int pieces_of(int tiles, int size)
{
    const int x = tiles + size - 1;
    const int q = (int)__fdividef((float)x, (float)size), r = x - q*size;
    return q + (r >= size ? 1 : 0) - (r < 0 ? 1 : 0);
}

// Shares that end where units end.  A worker whose share reaches into a second unit starts and
// ends twice, 2 us; it is cheaper to cut every unit into pieces of at most `size` tiles, a
// worker each, when there are workers for that with a size at or little above the even share
// (bf16, head 128, even shares against pieces: 32 units of 3000 positions 18.1 and 16.6 us, 144
// units of 3000 in e4m3 32.9 and 28.9; pieces half as large again as the share lose: 96 units
// of 2048, in L2, 19.2 and 22.7).  Working it out costs 0.5 us where nothing is gained: 8 units of
// 512 8.2 and 8.7, 96 of 2048 25.2 and 25.7.  Returns that size, or 0.  t0, t1: tiles of a unit of
// sequences lane, lane + 32.
template<int WARPS>
__device__ __forceinline__ int piece_size(int t0, int t1, int units_per_seq, int total,
        int workers)
{
    const int even = pieces_of(total, workers*WARPS), more = even + even/4;
    const int least = (int)__reduce_add_sync(0xffffffffu, pieces_of(t0, even*WARPS)
            + pieces_of(t1, even*WARPS))*units_per_seq;
    if(least <= workers)
    {
        return even*WARPS;
    }
    const int fewer = (int)__reduce_add_sync(0xffffffffu, pieces_of(t0, more*WARPS)
            + pieces_of(t1, more*WARPS))*units_per_seq;
    return fewer <= workers ? more*WARPS : 0;
}

// EXACT: the head size is DP.
template<typename T, bool E4M3, int DP, int MT, bool EXACT>
__global__ void __launch_bounds__(PagedTile<E4M3, DP>::WARPS*32, 1)
paged_decode_kernel(const PagedDecodeArgs a)
{
    using L = PagedTile<E4M3, DP>;
    using M = typename std::conditional<E4M3, __half, T>::type;      // operand format
    constexpr bool HALF = std::is_same<M, __half>::value;
    // A weight is exp2(score - reference).  The reference moves to LIFT below the largest score,
    // and only when a score passes that by more than SLACK: weights stay below
    // 2^(LIFT + SLACK) and most tiles do without a maximum.  bf16 has fp32's range.  fp16 has
    // not, so there the reference follows what the weights are multiplied with as well: for
    // 8-bit rows the score with the exponent of the value row's scale, and rows of zeros, which
    // may have all of the weight, do not count.  The largest weight times scale then is at least
    // 2^LIFT, and another counts down to 2^-34 of it.  The sums, in fp32, take all weights: they
    // may be DEEPEST binades above the reference, so that rows which count may be 2^80 smaller
    // than others that do not.  Whole binades here and in the scales: nothing rounds.
    constexpr float LIFT = HALF ? 10.0f : 0.0f, SLACK = HALF ? 5.5f : 4.0f, DEEPEST = 90.0f;
    // 8-bit values: accumulators count in units of 2^(vref - 127).  vref begins at the scale of
    // values around one, or of the first rows when those are more than SPREAD binades away, and
    // grows when a row is that much above it.
    constexpr int USUAL = 119, SPREAD = 60;
    constexpr float LOWEST = -3.0e38f;                   // no score yet
    constexpr int PARTS = HALF ? 2 : 3;                  // a weight's 16-bit pieces
    constexpr uint32_t LEAST = HALF ? 0x00010001u : 0x00800080u;     // 2^-24, 2^-126, twice
    constexpr int KSTEPS = DP/16, MBLK = L::MBLK, WARPS = L::WARPS, STAGES = L::STAGES;
    // Two tiles of heads are two chains already, and leave no registers for more (300 MB of 8-bit
    // rows of 128, group 16, a ragged batch of 64: 79 us, with two tiles of positions 91).
    constexpr int ABREAST = MT == 2 && L::ABREAST > 1 ? L::ABREAST/2 : L::ABREAST;
    constexpr int AHEAD = STAGES - ABREAST;              // tiles in flight or waiting
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int nv_s[WARPS][STAGES];
    __shared__ float top_s[WARPS][8], sum_s[WARPS][8];
    __shared__ int scan_s[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = lane >> 2, t = lane & 3;
    uint8_t *ring = smem + warp*STAGES*L::STAGE;
    float *merge = reinterpret_cast<float *>(smem + WARPS*STAGES*L::STAGE);
    const int D = EXACT ? DP : a.head, P = a.page_size;
    const int htiles = (a.group + 8*MT - 1)/(8*MT), HU = a.kv_heads*htiles;
    const int tpb = P/PD_TILE;

    // columns behind the head are never copied: zero for good
    if(D < DP)
    {
        uint4 *z = reinterpret_cast<uint4 *>(ring);
        for(int i = lane; i < STAGES*L::STAGE/16; i += 32)
        {
            z[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
    }

    chain_wait();

    // zeros for query heads g0, g0 + step, .. of unit (b, hu), which has nothing to attend to
    auto nothing = [&](int b, int hu, int g0, int step)
    {
        const int h0 = hu % htiles*8*MT, heads = min(8*MT, a.group - h0);
        for(int g = g0; g < heads; g += step)
        {
            const size_t qh = ((size_t)(hu/htiles)*a.group + h0 + g)*a.batch + b;
            for(int d = lane; d < D; d += 32)
            {
                ((T *)a.out)[qh*D + d] = from_f<T>(0.0f);
            }
            if(lane == 0 && a.lse_out)
            {
                a.lse_out[qh] = -CUDART_INF_F;
            }
        }
    };

    // ---- this worker's share: tiles [begin, end) of the row of all tiles, and the sequence b
    // it begins in, whose own tiles begin at seq_begin
    const int wpw = a.wpw, workers = gridDim.x*(WARPS/wpw);
    const int worker = blockIdx.x*(WARPS/wpw) + warp/wpw;
    int begin, end, b = 0, seq_begin = 0;
    int share = 0;                            // tiles of this worker's neighbours as well
    if(a.whole && (long long)a.batch*HU <= workers)
    {
        // a unit each at most: no need to know where the others' tiles are
        if(worker >= a.batch*HU)
        {
            return;
        }
        b = worker/HU;
        const int hu = worker - b*HU;
        const int nt = unit_tiles(a, checked_length(a.lengths, b, a.max_blocks*a.page_size,
                lane == 0 ? a.status : nullptr));
        begin = hu*nt;
        end = begin + nt;
        if(nt == 0)
        {
            nothing(b, hu, wpw > 1 ? warp : 0, wpw);
            return;                           // the whole worker
        }
    }
    else if(!a.whole && a.batch <= PD_BATCH)
    {
        // every warp finds the share by itself: no barrier before the first copies
        int tiles[2];                         // of a unit of sequences lane, lane + 32
#pragma unroll
        for(int i = 0; i < 2; ++i)
        {
            tiles[i] = 32*i + lane < a.batch ? unit_tiles(a, checked_length(a.lengths,
                    32*i + lane, a.max_blocks*a.page_size, blockIdx.x == 0 && warp == 0
                    ? a.status : nullptr)) : 0;
        }
        const int total = (int)__reduce_add_sync(0xffffffffu, (tiles[0] + tiles[1])*HU);
        const int size = wpw == 1 || total == 0 || a.batch*HU == 1 || a.batch*HU > workers ? 0
                : piece_size<WARPS>(tiles[0], tiles[1], HU, total, workers);
        const PagedShares sh = paged_shares<WARPS>(total, gridDim.x, wpw);
        // this worker's place in the row of all pieces, or of all tiles
        const int place = size > 0 ? worker
                : (int)min((long long)total, (long long)worker*sh.share);
        int before = 0, k = 32;               // where the sequence it is in begins, its lane
#pragma unroll
        for(int i = 0; i < 2; ++i)
        {
            const int mine = (size > 0 ? pieces_of(tiles[i], size) : tiles[i])*HU;
            int scan = mine;
#pragma unroll
            for(int o = 1; o < 32; o <<= 1)
            {
                const int up = __shfl_up_sync(0xffffffffu, scan, o);
                scan += lane >= o ? up : 0;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, before + scan > place);
            if(hit != 0u)
            {
                k = __ffs((int)hit) - 1;
                b = 32*i + k;
                before += __shfl_sync(0xffffffffu, scan - mine, k);
                break;
            }
            before += __shfl_sync(0xffffffffu, scan, 31);
        }
        if(k == 32)
        {
            return;                           // nothing left for this worker
        }
        if(size > 0)
        {
            const int nt = __shfl_sync(0xffffffffu, b < 32 ? tiles[0] : tiles[1], k);
            const int pieces = pieces_of(nt, size);
            const int hu = pieces_of(place - before + 1, pieces) - 1;
            share = ((nt + pieces - 1)/pieces + wpw - 1)/wpw*wpw;
            begin = min((hu + 1)*nt, hu*nt + (place - before - hu*pieces)*share);
            end = min((hu + 1)*nt, begin + share);
            if(begin >= end)
            {
                return;
            }
        }
        else
        {
            share = sh.share;
            seq_begin = before;
            begin = place;
            end = (int)min((long long)total, (long long)begin + sh.share);
        }
    }
    else
    {
        int *prefix = reinterpret_cast<int *>(merge);
        tile_prefix(a, HU, prefix, scan_s, blockIdx.x == 0);
        const int total = prefix[a.batch];
        if(a.whole)
        {
            // whole units, no joining: unit = sequence*HU + (kv head, head tile)
            const long long units = (long long)a.batch*HU;
            int x[2];
#pragma unroll
            for(int i = 0; i < 2; ++i)
            {
                const int u = (int)(units*(worker + i)/workers);
                const int ub = u/HU;
                x[i] = ub < a.batch ? prefix[ub] + (prefix[ub + 1] - prefix[ub])/HU*(u - ub*HU)
                        : total;
            }
            begin = x[0];
            end = x[1];
            const int u0 = (int)(units*worker/workers), u1 = (int)(units*(worker + 1)/workers);
            for(int u = u0 + (wpw > 1 ? warp : 0); u < u1; u += wpw)
            {
                const int ub = u/HU;
                if(prefix[ub + 1] == prefix[ub])
                {
                    nothing(ub, u - ub*HU, 0, 1);
                }
            }
        }
        else
        {
            const PagedShares sh = paged_shares<WARPS>(total, gridDim.x, wpw);
            share = sh.share;
            begin = (int)min((long long)total, (long long)worker*sh.share);
            end = (int)min((long long)total, (long long)begin + sh.share);
        }
        if(begin < end)
        {
            int lo = 0, hi = a.batch;         // prefix[lo] <= begin < prefix[hi]
            while(hi - lo > 1)
            {
                const int mid = (lo + hi) >> 1;
                if(prefix[mid] <= begin) lo = mid;
                else hi = mid;
            }
            b = lo;
        }
        seq_begin = prefix[b];
        __syncthreads();                      // the prefix sums give way to the merge buffer
        if(begin >= end)
        {
            return;                           // the whole block when wpw > 1: same share
        }
    }

    // ---- issuing side: runs STAGES - 1 tiles ahead of the consuming side
    const int step = wpw, slot0 = wpw > 1 ? warp : 0;
    int ib = b, ix = begin + slot0 - seq_begin;          // next tile, counted inside sequence ib
    int ileft = end - begin > slot0 ? (end - begin - slot0 + step - 1)/step : 0;
    int ilen = held_len(a, ib), int_ = unit_tiles(a, ilen);
    int ipos = 32;                                       // used up: look up at once
    uint32_t look = 0;                                   // first row/16 << 5 | rows filled
    const int row_bytes = EXACT ? L::ROW_BYTES : D*(E4M3 ? 1 : (int)sizeof(T));
    const int chunks = row_bytes/16;
    constexpr int RPP = 32/L::CHUNKS > 0 ? 32/L::CHUNKS : 1;     // rows a warp copies at once
    const int crow = lane/L::CHUNKS, cchunk = lane % L::CHUNKS;
    const uint8_t *k_lane = (const uint8_t *)a.k_pages + crow*row_bytes + cchunk*16;
    const uint8_t *v_lane = (const uint8_t *)a.v_pages + crow*row_bytes + cchunk*16;

    auto issue = [&](int stage)
    {
        if(ileft > 0)
        {
            if(ix >= int_*HU)
            {
                while(ix >= int_*HU)
                {
                    ix -= int_*HU;
                    ++ib;
                    ilen = held_len(a, ib);
                    int_ = unit_tiles(a, ilen);
                }
                ipos = 32;
            }
            if(ipos == 32)
            {
                // pages of this warp's next 32 tiles in the sequence
                ipos = 0;
                look = 0;
                const long long x = ix + (long long)lane*step;
                if(x < (long long)int_*HU && lane < ileft)
                {
                    const int unit = (int)x/int_, j = (int)x - unit*int_, kvh = unit/htiles;
                    const int li = j/tpb, sub = (j - li*tpb)*PD_TILE;
                    int block = li;
                    if(a.selected)
                    {
                        bool bad = false;
                        block = held_block(a.selected[((size_t)kvh*a.batch + ib)*a.num_selected
                                + li], blocks_of(ilen, P), a.max_blocks, bad);
                        if(bad)
                        {
                            report(a.status, NNTILE_B200_PAGED_BAD_BLOCK);
                        }
                    }
                    if(block >= 0)
                    {
                        const int left = ilen - block*P - sub;
                        const int page = left > 0 ? checked_page(a.block_table
                                + (size_t)ib*a.max_blocks, block, a.num_pages, a.status) : -1;
                        if(page >= 0)
                        {
                            const uint32_t row = ((uint32_t)page*(uint32_t)a.kv_heads + kvh)
                                    *(uint32_t)P + sub;
                            look = row/PD_TILE << 5 | (uint32_t)min(left, PD_TILE);
                        }
                    }
                }
            }
            const uint32_t here = __shfl_sync(0xffffffffu, look, ipos);
            const int nv = (int)(here & 31u);
            const uint32_t row = (here >> 5)*PD_TILE;
            if(lane == 0)
            {
                nv_s[warp][stage] = nv;
            }
            const uint32_t dst = smem_addr(ring + stage*L::STAGE);
            const uint8_t *ks = k_lane + (size_t)row*row_bytes;
            const uint8_t *vs = v_lane + (size_t)row*row_bytes;
            if(nv == PD_TILE)
            {
                if(EXACT || cchunk < chunks)
                {
#pragma unroll
                    for(int i = 0; i < PD_TILE/RPP; ++i)
                    {
                        copy16(dst + L::offset(crow + i*RPP, cchunk, E4M3),
                                ks + i*RPP*row_bytes, 16);
                        copy16(dst + L::KV_BYTES + L::offset(crow + i*RPP, cchunk, false),
                                vs + i*RPP*row_bytes, 16);
                    }
                }
            }
            else if(EXACT || cchunk < chunks)
            {
                // rows behind the length, and all of a tile without a page: zeros
#pragma unroll
                for(int i = 0; i < PD_TILE/RPP; ++i)
                {
                    const int bytes = crow + i*RPP < nv ? 16 : 0;
                    copy16(dst + L::offset(crow + i*RPP, cchunk, E4M3), ks + i*RPP*row_bytes,
                            bytes);
                    copy16(dst + L::KV_BYTES + L::offset(crow + i*RPP, cchunk, false),
                            vs + i*RPP*row_bytes, bytes);
                }
            }
            if(E4M3 && lane < 2)
            {
                copy16(dst + 2*L::KV_BYTES + lane*PD_TILE,
                        (lane == 0 ? a.k_scales : a.v_scales) + row, nv > 0 ? 16 : 0);
            }
            ++ipos;
            ix += step;
            --ileft;
        }
        copy_commit();
    };
#pragma unroll 1
    for(int s = 0; s < AHEAD; ++s)
    {
        issue(s);                                        // once in the code: it is long
    }

    // ---- consuming side, unit by unit
    int stage = 0;
    int seq_len = held_len(a, b);
    int nt = unit_tiles(a, seq_len);
    int hu = (begin - seq_begin)/nt;
    int x = begin;                                       // first tile of the segment
    int unit_begin = seq_begin + hu*nt;
    int mine = begin + slot0;                            // this warp's next tile
    while(x < end)
    {
        const int unit_end = unit_begin + nt;
        const int seg_end = min(end, unit_end);
        const int kvh = hu/htiles, h0 = (hu - kvh*htiles)*8*MT;
        const int heads = min(8*MT, a.group - h0);

        uint32_t qa[MT][KSTEPS][2];
        float qscale[MT][2];                             // of heads 2t, 2t + 1
#pragma unroll
        for(int m = 0; m < MT; ++m)
        {
            const int g = 8*m + n;
            const T *qr = (const T *)a.q + (((size_t)kvh*a.group + h0 + min(g, heads - 1))
                    *a.batch + b)*D;
            qscale[m][0] = qscale[m][1] = a.scale_log2;
#pragma unroll
            for(int k = 0; k < KSTEPS; ++k)
#pragma unroll
                for(int x2 = 0; x2 < 2; ++x2)
                {
                    // head elements of this lane's operand word: in order for 16-bit rows; for
                    // codes a lane's 16-byte piece t + 4j feeds four steps, four codes each
                    const int d = E4M3 ? 16*(t + 4*(k >> 2)) + 4*(k & 3) + 2*x2
                            : 16*k + 8*x2 + 2*t;
                    qa[m][k][x2] = d < D && g < heads
                            ? *reinterpret_cast<const uint32_t *>(qr + d) : 0u;
                }
            if(E4M3 && !std::is_same<T, __half>::value)
            {
                // bf16 queries as fp16 operands: a power of two brings the row's largest element
                // to [2^14, 2^15); what fp16 then loses is below 2^-38 of it
                float amax = 0.0f;
#pragma unroll
                for(int k = 0; k < KSTEPS; ++k)
#pragma unroll
                    for(int x2 = 0; x2 < 2; ++x2)
                    {
                        const float2 f = unpack2<T>(qa[m][k][x2]);
                        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int e = (int)(__float_as_uint(amax) >> 23);        // 0 and 255: as it is
                const int up = e == 255 ? 0 : max(-113, min(126, 141 - e));
                const float lift = __uint_as_float((uint32_t)(127 + up) << 23);
                const float undo = __uint_as_float((uint32_t)(127 - up) << 23);
                qscale[m][0] *= __shfl_sync(0xffffffffu, undo, 8*t);         // lane of head 2t
                qscale[m][1] *= __shfl_sync(0xffffffffu, undo, 8*t + 4);
#pragma unroll
                for(int k = 0; k < KSTEPS; ++k)
#pragma unroll
                    for(int x2 = 0; x2 < 2; ++x2)
                    {
                        const float2 f = unpack2<T>(qa[m][k][x2]);
                        qa[m][k][x2] = pack2<__half>(f.x*lift, f.y*lift);
                    }
            }
        }
        // the sum of weights is sum - over
        float acc[MT][MBLK][4], top[MT][2], sum[MT][2], over[MT][2];
#pragma unroll
        for(int m = 0; m < MT; ++m)
        {
            top[m][0] = top[m][1] = LOWEST;
            sum[m][0] = sum[m][1] = over[m][0] = over[m][1] = 0.0f;
#pragma unroll
            for(int i = 0; i < MBLK; ++i)
#pragma unroll
                for(int r = 0; r < 4; ++r)
                    acc[m][i][r] = 0.0f;
        }
        int vref = USUAL;

        // N tiles at once.  Keys and values are the 16-row operand, the query heads the 8
        // columns: this lane holds the scores of positions n and n + 8 of a tile for heads 2t
        // and 2t + 1, in the order [2*(position >= 8) + (head odd)].  FULL: all 16 rows of every
        // tile are filled.
        auto process = [&](auto tiles, auto filled)
        {
            constexpr int N = decltype(tiles)::value;
            constexpr bool FULL = decltype(filled)::value;
            const uint8_t *st[N];
            int nv[N];
            int to = stage + AHEAD;
            to -= to >= STAGES ? STAGES : 0;
#pragma unroll 1
            for(int j = 0; j < N; ++j)
            {
                issue(to);
                to = to + 1 == STAGES ? 0 : to + 1;
            }
#pragma unroll
            for(int j = 0; j < N; ++j)
            {
                st[j] = ring + stage*L::STAGE;
                nv[j] = FULL ? PD_TILE : nv_s[warp][stage];
                stage = stage + 1 == STAGES ? 0 : stage + 1;
            }
            if(!FULL && nv[0] == 0)
            {
                return;                                  // N = 1
            }
            // ---- scores, in two sums of every other step: half as long a chain
            float s[MT][N][2][4];
#pragma unroll
            for(int m = 0; m < MT; ++m)
#pragma unroll
                for(int j = 0; j < N; ++j)
#pragma unroll
                    for(int r = 0; r < 4; ++r)
                        s[m][j][0][r] = s[m][j][1][r] = 0.0f;
            if(!E4M3)
            {
                const int r = lane & 15, col = lane >> 4;
#pragma unroll
                for(int k = 0; k < KSTEPS; ++k)
#pragma unroll
                    for(int j = 0; j < N; ++j)
                    {
                        uint32_t ka[4];
                        ldmatrix4(ka, smem_addr(st[j] + L::offset(r, 2*k + col, false)));
#pragma unroll
                        for(int m = 0; m < MT; ++m)
                        {
                            mma16<M>(s[m][j][k & 1], ka[0], ka[1], ka[2], ka[3], qa[m][k][0],
                                    qa[m][k][1]);
                        }
                    }
            }
            else
            {
#pragma unroll
                for(int c4 = 0; c4 < DP/64; ++c4)
                {
                    uint4 kc[N][2];
#pragma unroll
                    for(int j = 0; j < N; ++j)
#pragma unroll
                        for(int h = 0; h < 2; ++h)
                        {
                            kc[j][h] = *reinterpret_cast<const uint4 *>(st[j]
                                    + L::offset(8*h + n, t + 4*c4, true));
                        }
#pragma unroll
                    for(int w = 0; w < 4; ++w)
#pragma unroll
                        for(int j = 0; j < N; ++j)
                        {
                            const uint32_t c = word4(kc[j][0], w), d = word4(kc[j][1], w);
                            const uint32_t a0 = e4m3x2_to_half2(c & 0xFFFFu);
                            const uint32_t a1 = e4m3x2_to_half2(d & 0xFFFFu);
                            const uint32_t a2 = e4m3x2_to_half2(c >> 16);
                            const uint32_t a3 = e4m3x2_to_half2(d >> 16);
#pragma unroll
                            for(int m = 0; m < MT; ++m)
                            {
                                mma16<M>(s[m][j][w & 1], a0, a1, a2, a3, qa[m][4*c4 + w][0],
                                        qa[m][4*c4 + w][1]);
                            }
                        }
                }
            }
            // factors of the scores, by position and head; what is over `limit` moves the reference
            float factor[MT][N][2][2], limit[N][2];
            int vbyte[N][2];
            bool moved = false;
#pragma unroll
            for(int j = 0; j < N; ++j)
#pragma unroll
                for(int h = 0; h < 2; ++h)
                {
                    float kscale = 1.0f;
                    limit[j][h] = LIFT + SLACK;
                    if(E4M3)
                    {
                        const uint8_t *sc = st[j] + 2*L::KV_BYTES + 8*h + n;
                        kscale = __uint_as_float((uint32_t)sc[0] << 23);
                        // the scale of a row behind the length may be anything: keep it out
                        vbyte[j][h] = FULL || 8*h + n < nv[j] ? (int)sc[PD_TILE] : vref;
                        moved = moved || vbyte[j][h] > vref + SPREAD;
                        limit[j][h] = fminf(limit[j][h] - (float)(vbyte[j][h] - vref), DEEPEST);
                    }
#pragma unroll
                    for(int m = 0; m < MT; ++m)
#pragma unroll
                        for(int y = 0; y < 2; ++y)
                            factor[m][j][h][y] = E4M3 ? qscale[m][y]*kscale : qscale[m][y];
                }
            // d = score - reference, in the place of the first sum
#pragma unroll
            for(int m = 0; m < MT; ++m)
#pragma unroll
                for(int j = 0; j < N; ++j)
#pragma unroll
                    for(int r = 0; r < 4; ++r)
                    {
                        s[m][j][1][r] += s[m][j][0][r];
                        float d = fmaf(s[m][j][1][r], factor[m][j][r >> 1][r & 1],
                                -top[m][r & 1]);
                        if(!FULL)
                        {
                            d = 8*(r >> 1) + n < nv[j] ? d : -CUDART_INF_F;
                        }
                        s[m][j][0][r] = d;
                        moved = moved || d > limit[j][r >> 1];
                    }
            if(__any_sync(0xffffffffu, moved))
            {
                // rows that are zero, scales far from vref: all that is unusual comes first
                bool odd = false;
                uint32_t blank = 0u;                     // bit 2j + h: the value row is zero
                float back = 1.0f, least[MT][2];         // of accumulators, for references
                if(HALF)
                {
                    constexpr uint32_t SIZE = E4M3 ? 0x7F7F7F7Fu : 0x7FFF7FFFu;
#pragma unroll
                    for(int j = 0; j < N; ++j)
#pragma unroll
                        for(int h = 0; h < 2; ++h)
                        {
                            // four words of a row first, seldom are they zero
                            const uint32_t some = *reinterpret_cast<const uint32_t *>(st[j]
                                    + L::KV_BYTES + L::offset(8*h + n, t, false)) & SIZE;
                            odd = odd || some == 0u
                                    || (E4M3 && abs(vbyte[j][h] - vref) > SPREAD);
                        }
                    odd = __any_sync(0xffffffffu, odd);
                }
#pragma unroll
                for(int m = 0; m < MT; ++m)
#pragma unroll
                    for(int y = 0; y < 2; ++y)
                        least[m][y] = top[m][y];
                if(HALF && __builtin_expect(odd, 0))
                {
                    constexpr uint32_t SIZE = E4M3 ? 0x7F7F7F7Fu : 0x7FFF7FFFu;
#pragma unroll
                    for(int j = 0; j < N; ++j)
#pragma unroll
                        for(int h = 0; h < 2; ++h)
                        {
                            uint32_t some = 0u;          // in this lane's quarter of the row
#pragma unroll
                            for(int c = 0; c < L::CHUNKS; c += 4)
                            {
                                const uint4 v = *reinterpret_cast<const uint4 *>(st[j]
                                        + L::KV_BYTES + L::offset(8*h + n, t + c, false));
                                some |= (v.x | v.y | v.z | v.w) & SIZE;
                            }
                            blank |= some == 0u ? 1u << (2*j + h) : 0u;
                        }
                    blank &= __shfl_xor_sync(0xffffffffu, blank, 1);
                    blank &= __shfl_xor_sync(0xffffffffu, blank, 2);
                    int grown = 0;
                    if(E4M3)
                    {
                        bool fresh = true;               // nothing is counted in vref yet
#pragma unroll
                        for(int m = 0; m < MT; ++m)
                        {
                            fresh = fresh && top[m][0] == LOWEST && top[m][1] == LOWEST;
                        }
                        fresh = __all_sync(0xffffffffu, fresh);
                        int vtop = 0;
#pragma unroll
                        for(int j = 0; j < N; ++j)
#pragma unroll
                            for(int h = 0; h < 2; ++h)
                                if((blank >> (2*j + h) & 1u) == 0u)
                                {
                                    vtop = max(vtop, vbyte[j][h]);
                                }
                        vtop = __reduce_max_sync(0xffffffffu, vtop);
                        if(vtop > 0 && (fresh || vtop > vref + SPREAD))
                        {
                            grown = fresh ? 0 : vtop - vref;
                            back = ex2(-(float)grown);
                            vref = vtop;
                        }
                    }
#pragma unroll
                    for(int j = 0; j < N; ++j)
#pragma unroll
                        for(int h = 0; h < 2; ++h)
                        {
                            const bool zero = (blank >> (2*j + h) & 1u) != 0u;
                            if(E4M3)
                            {
                                vbyte[j][h] = zero ? vref : vbyte[j][h];
                                limit[j][h] = LIFT + SLACK - (float)(vbyte[j][h] - vref);
                            }
                            limit[j][h] = zero ? CUDART_INF_F : limit[j][h];
                        }
                    // What vref grows by the references give way, as far as the sums, which are
                    // in fp32, have room for.
#pragma unroll
                    for(int m = 0; m < MT; ++m)
#pragma unroll
                        for(int y = 0; y < 2; ++y)
                        {
                            float all = -CUDART_INF_F, most = sum[m][y];
#pragma unroll
                            for(int j = 0; j < N; ++j)
#pragma unroll
                                for(int h = 0; h < 2; ++h)
                                    if(FULL || 8*h + n < nv[j])
                                    {
                                        all = fmaxf(all, s[m][j][1][2*h + y]*factor[m][j][h][y]);
                                    }
#pragma unroll
                            for(int o = 4; o < 32; o <<= 1)
                            {
                                all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
                                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                            }
                            const float give = fminf((float)grown, 100.0f
                                    - fmaxf(0.0f, ceilf(__log2f(most))));
                            least[m][y] = fmaxf(top[m][y] - give, ceilf(all) - DEEPEST);
                        }
                }
#pragma unroll
                for(int m = 0; m < MT; ++m)
                {
                    float f[2];
#pragma unroll
                    for(int y = 0; y < 2; ++y)
                    {
                        float ntop = -CUDART_INF_F;
#pragma unroll
                        for(int j = 0; j < N; ++j)
#pragma unroll
                            for(int h = 0; h < 2; ++h)
                                if(FULL || 8*h + n < nv[j])
                                {
                                    ntop = fmaxf(ntop, fmaf(s[m][j][1][2*h + y],
                                            factor[m][j][h][y], HALF ? -limit[j][h] : 0.0f));
                                }
#pragma unroll
                        for(int o = 4; o < 32; o <<= 1)
                        {
                            ntop = fmaxf(ntop, __shfl_xor_sync(0xffffffffu, ntop, o));
                        }
                        // fp16: LIFT below what is over the limit, on a whole binade
                        ntop = fmaxf(least[m][y], HALF ? floorf(ntop + SLACK) : ntop - LIFT);
                        const float shrink = ntop == top[m][y] ? 1.0f : ex2(top[m][y] - ntop);
                        top[m][y] = ntop;
                        sum[m][y] *= shrink;
                        over[m][y] *= shrink;
                        f[y] = E4M3 ? shrink*back : shrink;
#pragma unroll
                        for(int j = 0; j < N; ++j)
#pragma unroll
                            for(int h = 0; h < 2; ++h)
                                if(FULL || 8*h + n < nv[j])
                                {
                                    s[m][j][0][2*h + y] = fmaf(s[m][j][1][2*h + y],
                                            factor[m][j][h][y], -ntop);
                                }
                    }
#pragma unroll
                    for(int i = 0; i < MBLK; ++i)
#pragma unroll
                        for(int r = 0; r < 4; ++r)
                            acc[m][i][r] *= f[r & 1];
                }
                if(HALF && __builtin_expect(odd, 0))
                {
                    // weights of rows of zeros: only in the sum
#pragma unroll
                    for(int m = 0; m < MT; ++m)
#pragma unroll
                        for(int j = 0; j < N; ++j)
#pragma unroll
                            for(int r = 0; r < 4; ++r)
                                if((blank >> (2*j + (r >> 1)) & 1u) != 0u)
                                {
                                    sum[m][r & 1] += ex2(s[m][j][0][r]);
                                    s[m][j][0][r] = -CUDART_INF_F;
                                }
                }
            }
            // ---- weights, in 16-bit parts, as the 8-column operand of the second product
            uint32_t pb[MT][N][PARTS][2];                // part, positions >= 8
            float more[MT][2];                           // to the sums
#pragma unroll
            for(int m = 0; m < MT; ++m)
                more[m][0] = more[m][1] = 0.0f;
#pragma unroll
            for(int j = 0; j < N; ++j)
#pragma unroll
                for(int h = 0; h < 2; ++h)
                {
                    // 2^(scale of the row - scale of the accumulators), 0 when far below
                    const float rel = E4M3 ? __uint_as_float((uint32_t)max(vbyte[j][h] - vref + 127,
                            0) << 23) : 1.0f;
#pragma unroll
                    for(int m = 0; m < MT; ++m)
                    {
                        float p[2];
#pragma unroll
                        for(int y = 0; y < 2; ++y)
                        {
                            p[y] = ex2(s[m][j][0][2*h + y]);
                            more[m][y] += p[y];
                            if(E4M3)
                            {
                                p[y] *= rel;
                            }
                        }
                        // Values of T may be infinite, and 0 * inf is NaN: all parts but the last
                        // are cut off, and those after the first raised to LEAST where they
                        // are less, so that all are positive where the weight is (from LEAST on).
                        uint32_t up = 0u;
#pragma unroll
                        for(int part = 0; part < PARTS; ++part)
                        {
                            uint32_t w = E4M3 || part == PARTS - 1 ? pack2<M>(p[0], p[1])
                                    : cut2<M>(p[0], p[1]);
                            if(part == 0)
                            {
                                up = w;
                            }
                            else if(!E4M3)
                            {
                                w = max2<M>(w, min2<M>(up, LEAST));
                            }
                            pb[m][j][part][h] = transpose8x8(w);
                            const float2 kept = unpack2<M>(w);
                            p[0] -= kept.x;
                            p[1] -= kept.y;
                        }
                    }
                }
            // Like weights, thousands of them, would all round the same way (2^-14 of the sum of
            // 131072): what a sum takes too much is kept and taken off again.
#pragma unroll
            for(int m = 0; m < MT; ++m)
            {
                float part[2], next[2];
                minus2(part, more[m], over[m]);
                plus2(next, sum[m], part);
                minus2(over[m], next, sum[m]);
                minus2(over[m], over[m], part);
                sum[m][0] = next[0];
                sum[m][1] = next[1];
            }
            // ---- O += P V
#pragma unroll
            for(int j = 0; j < N; ++j)
            {
                const uint8_t *sv = st[j] + L::KV_BYTES;
                if(!E4M3)
                {
                    const int r = (lane & 7) + ((lane >> 4) << 3), col = (lane >> 3) & 1;
                    // Four blocks of columns side by side, each a chain of PARTS products (300 MB of
                    // heads of 256, group 16: 82 us, one after the other 92).
                    constexpr int SIDE = 4;
#pragma unroll
                    for(int i0 = 0; i0 < MBLK; i0 += SIDE)
                    {
                        uint32_t va[SIDE][4];
                        float o[SIDE][MT][4];
#pragma unroll
                        for(int i = 0; i < SIDE; ++i)
                            ldmatrix4_trans(va[i], smem_addr(sv + L::offset(r, 2*(i0 + i) + col,
                                    false)));
                        // The instruction cuts its sums off, always downwards in size; over
                        // a long chain that adds up (means of 131072 fp16 positions: one in
                        // three not the nearest number).  So a tile's sum, smallest parts
                        // first, is added as an ordinary fp32 number (64 sequences of 8192:
                        // 325 -> 331 us, 37 ragged ones in 8 bits 134 -> 137).
#pragma unroll
                        for(int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                            for(int i = 0; i < SIDE; ++i)
#pragma unroll
                                for(int m = 0; m < MT; ++m)
                                {
                                    if(part == PARTS - 1)
                                    {
                                        o[i][m][0] = o[i][m][1] = o[i][m][2] = o[i][m][3] = 0.0f;
                                    }
                                    mma16<M>(o[i][m], va[i][0], va[i][1], va[i][2], va[i][3],
                                            pb[m][j][part][0], pb[m][j][part][1]);
                                }
#pragma unroll
                        for(int i = 0; i < SIDE; ++i)
#pragma unroll
                            for(int m = 0; m < MT; ++m)
                                add4(acc[m][i0 + i], o[i][m]);
                    }
                }
                else
                {
                    constexpr int VW = DP == 64 ? 2 : 4;     // words of a lane's piece of a row
#pragma unroll
                    for(int q4 = 0; q4 < (DP + 127)/128; ++q4)
                    {
                        uint32_t vw[4][VW];
#pragma unroll
                        for(int role = 0; role < 4; ++role)
                        {
                            const int r = 2*t + (role & 1) + 8*(role >> 1);
                            if(DP == 64)
                            {
                                const uint2 v = *reinterpret_cast<const uint2 *>(sv
                                        + L::offset(r, n >> 1, false) + 8*(n & 1));
                                vw[role][0] = v.x;
                                vw[role][1] = v.y;
                            }
                            else
                            {
                                const uint4 v = *reinterpret_cast<const uint4 *>(sv
                                        + L::offset(r, n + 8*q4, false));
                                vw[role][0] = v.x;
                                vw[role][1] = v.y;
                                vw[role][VW - 2] = DP == 64 ? v.x : v.z;
                                vw[role][VW - 1] = DP == 64 ? v.y : v.w;
                            }
                        }
#pragma unroll
                        for(int w = 0; w < VW; ++w)
#pragma unroll
                            for(int pair = 0; pair < 2; ++pair)
                            {
                                // codes 2*pair and 2*pair + 1 of the word, positions 2t, 2t + 1
                                const uint32_t sel = pair ? 0x7362u : 0x5140u;
                                const uint32_t lo = __byte_perm(vw[0][w], vw[1][w], sel);
                                const uint32_t hi = __byte_perm(vw[2][w], vw[3][w], sel);
                                const uint32_t a0 = e4m3x2_to_half2(lo & 0xFFFFu);
                                const uint32_t a1 = e4m3x2_to_half2(lo >> 16);
                                const uint32_t a2 = e4m3x2_to_half2(hi & 0xFFFFu);
                                const uint32_t a3 = e4m3x2_to_half2(hi >> 16);
                                const int i = 8*q4 + 2*w + pair;
#pragma unroll
                                for(int m = 0; m < MT; ++m)
                                {
                                    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                    for(int part = PARTS - 1; part >= 0; --part)
                                        mma16<M>(o, a0, a1, a2, a3, pb[m][j][part][0],
                                                pb[m][j][part][1]);
                                    add4(acc[m][i], o);
                                }
                            }
                    }
                }
            }
        };
        while(mine < seg_end)
        {
            copy_wait<AHEAD - ABREAST>();
            // every lane's copies are there, and what was consumed last is free
            __syncwarp();
            bool full = ABREAST > 1 && mine + (ABREAST - 1)*step < seg_end;
            int at = stage;
#pragma unroll
            for(int j = 0; j < ABREAST; ++j)
            {
                full = full && nv_s[warp][at] == PD_TILE;
                at = at + 1 == STAGES ? 0 : at + 1;
            }
            if(ABREAST == 1)
            {
                full = nv_s[warp][stage] == PD_TILE;
            }
            if(full)
            {
                mine += ABREAST*step;
                process(std::integral_constant<int, ABREAST>(), std::true_type());
            }
            else
            {
                mine += step;
                process(std::integral_constant<int, 1>(), std::false_type());
            }
        }

        // ---- end of the segment: join the warps of the worker, then write the unit, or
        // this share's part of it
        const bool complete = x == unit_begin && seg_end == unit_end;
        const int part = 2*worker + (x == unit_begin ? 1 : 0);
        if(share > 0 && x == unit_begin && lane == 0 && slot0 == 0)
        {
            // the others of this unit follow, a share each
            a.spans[b*HU + hu] = make_int2(worker, worker + (complete ? 0
                    : (unit_end - end + share - 1)/share));
        }
        const float vscale = E4M3 ? scale_value((uint32_t)vref) : 1.0f;
#pragma unroll
        for(int m = 0; m < MT; ++m)
        {
#pragma unroll
            for(int y = 0; y < 2; ++y)
            {
                sum[m][y] -= over[m][y];
#pragma unroll
                for(int o = 4; o < 32; o <<= 1)
                {
                    sum[m][y] += __shfl_xor_sync(0xffffffffu, sum[m][y], o);
                }
            }
            if(HALF)
            {
                // sums to [1, 2): what is joined by its reference has no need of more range
                float f[2];
#pragma unroll
                for(int y = 0; y < 2; ++y)
                {
                    const int e = sum[m][y] == 0.0f ? 0
                            : max(-120, min(120, (int)(__float_as_uint(sum[m][y]) >> 23) - 127));
                    f[y] = __uint_as_float((uint32_t)(127 - e) << 23);
                    sum[m][y] *= f[y];
                    f[y] *= vscale;
                    top[m][y] += (float)e;
                }
#pragma unroll
                for(int i = 0; i < MBLK; ++i)
#pragma unroll
                    for(int r = 0; r < 4; ++r)
                        acc[m][i][r] *= f[r & 1];
            }
            if(wpw > 1)
            {
                if(n == 0)
                {
#pragma unroll
                    for(int y = 0; y < 2; ++y)
                    {
                        top_s[warp][2*t + y] = top[m][y];
                        sum_s[warp][2*t + y] = sum[m][y];
                    }
                }
                float big[2], den[2], wgt[WARPS][2];
                constexpr int ROUND = MBLK/L::ROUNDS;        // blocks a round
                float *mw = merge + warp*ROUND*128;
#pragma unroll
                for(int q = 0; q < L::ROUNDS; ++q)
                {
#pragma unroll
                    for(int i = 0; i < ROUND; ++i)
#pragma unroll
                        for(int r = 0; r < 4; ++r)
                            mw[(4*i + r)*32 + lane] = acc[m][q*ROUND + i][r];
                    __syncthreads();
                    if(q == 0)
                    {
#pragma unroll
                        for(int y = 0; y < 2; ++y)
                        {
                            big[y] = -CUDART_INF_F;
                            den[y] = 0.0f;
#pragma unroll
                            for(int w = 0; w < WARPS; ++w)
                            {
                                big[y] = fmaxf(big[y], top_s[w][2*t + y]);
                            }
                            const float ref = big[y] == -CUDART_INF_F ? 0.0f : big[y];
#pragma unroll
                            for(int w = 0; w < WARPS; ++w)
                            {
                                wgt[w][y] = ex2(top_s[w][2*t + y] - ref);
                                den[y] = fmaf(wgt[w][y], sum_s[w][2*t + y], den[y]);
                            }
                        }
                    }
                    // every warp joins its share of the blocks, same lanes, same heads; with
                    // fewer blocks than warps the upper ones have none
                    constexpr int MY = (ROUND + WARPS - 1)/WARPS;
#pragma unroll
                    for(int k = 0; k < MY; ++k)
                    {
                        const int i = warp*MY + k;
                        if(i < ROUND)
                        {
                            float z[4];
#pragma unroll
                            for(int r = 0; r < 4; ++r)
                            {
                                z[r] = 0.0f;
#pragma unroll
                                for(int w = 0; w < WARPS; ++w)
                                {
                                    z[r] = fmaf(wgt[w][r & 1],
                                            merge[(w*ROUND*4 + 4*i + r)*32 + lane], z[r]);
                                }
                            }
                            write_part<T, E4M3, DP, MT>(a, complete, part, m, lane,
                                    q*ROUND + i, z, den, kvh, h0, heads, b);
                        }
                    }
                    if(q + 1 < L::ROUNDS)
                    {
                        __syncthreads();
                    }
                }
                if(warp == 0 && n == 0)
                {
#pragma unroll
                    for(int y = 0; y < 2; ++y)
                    {
                        write_sums<MT>(a, complete, part, m, 2*t + y, big[y], den[y], kvh, h0,
                                heads, b);
                    }
                }
                __syncthreads();
            }
            else
            {
#pragma unroll
                for(int i = 0; i < MBLK; ++i)
                {
                    write_part<T, E4M3, DP, MT>(a, complete, part, m, lane, i, acc[m][i], sum[m],
                            kvh, h0, heads, b);
                }
                if(n == 0)
                {
#pragma unroll
                    for(int y = 0; y < 2; ++y)
                    {
                        write_sums<MT>(a, complete, part, m, 2*t + y, top[m][y], sum[m][y], kvh,
                                h0, heads, b);
                    }
                }
            }
        }

        // ---- next unit
        x = seg_end;
        unit_begin = unit_end;
        if(++hu == HU && x < end)
        {
            hu = 0;
            do
            {
                ++b;
                nt = unit_tiles(a, held_len(a, b));
            }
            while(nt == 0);
        }
    }
}

// Joins the parts of the units that fell into several shares, and answers those with
// nothing to attend to.  A piece is 128 columns of a unit's heads, four neighbouring ones a
// lane; `wpp` warps share the parts of a piece and meet in shared memory: one warp while
// units are many and their parts few, up to 32 when a few units have many parts each.
__host__ __device__ inline int join_pieces(int heads, int dp)
{
    return (heads*dp + 127)/128;
}

struct JoinState                         // four values of a head, not yet divided by the sum
{
    float top, sum;
    float4 o;
};

// N more parts at once: one maximum, and weights that do not wait for one another.
template<int N>
__device__ __forceinline__ void join_add(JoinState &s, const float2 (&ts)[N], const float4 (&o)[N])
{
    float top = s.top;
#pragma unroll
    for(int u = 0; u < N; ++u)
    {
        top = fmaxf(top, ts[u].x);
    }
    const float ref = top == -CUDART_INF_F ? 0.0f : top, x = ex2(s.top - ref);
    s.top = top;
    s.sum *= x;
    s.o.x *= x;
    s.o.y *= x;
    s.o.z *= x;
    s.o.w *= x;
#pragma unroll
    for(int u = 0; u < N; ++u)
    {
        const float y = ex2(ts[u].x - ref);
        s.sum = fmaf(ts[u].y, y, s.sum);
        s.o.x = fmaf(o[u].x, y, s.o.x);
        s.o.y = fmaf(o[u].y, y, s.o.y);
        s.o.z = fmaf(o[u].z, y, s.o.z);
        s.o.w = fmaf(o[u].w, y, s.o.w);
    }
}

template<typename T, bool E4M3, int DP, int MT, int JOIN_WARPS>
__global__ void __launch_bounds__(JOIN_WARPS*32)
paged_join_kernel(const PagedDecodeArgs a, int workers, int wpp)
{
    const int pieces = join_pieces(min(8*MT, a.group), DP);
    __shared__ float2 sums_s[JOIN_WARPS][2];             // of lanes 0-15 and 16-31: one head each
    __shared__ float4 o_s[JOIN_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int htiles = (a.group + 8*MT - 1)/(8*MT), HU = a.kv_heads*htiles;
    const int id = (blockIdx.x*JOIN_WARPS + warp)/wpp;
    const int unit = id/pieces, piece = id - unit*pieces;
    const int b = min(unit/HU, a.batch - 1), hu = unit - b*HU;
    const bool some = unit < a.batch*HU && held_len(a, b) > 0;
    const int m = piece*128/(8*DP), off = piece*128 - m*8*DP + 4*lane;   // in the part's values
    const int head = off/DP, col = off - head*DP;
    const int kvh = hu/htiles, g = (hu - kvh*htiles)*8*MT + 8*m + head;
    chain_wait();
    const int2 span = some ? a.spans[unit] : make_int2(0, -1);
    const int first = max(span.x, 0), last = min(span.y, workers - 1);
    // one worker had it all and wrote it, or there is no such head, or (the last block) unit
    const bool none = first == last || g >= a.group || unit >= a.batch*HU;
    JoinState s = {-CUDART_INF_F, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    if(!none)
    {
        // the first share holds the unit's beginning in its second part, the others in their
        // first
        const int parts = last - first + 1;
        for(int i0 = warp % wpp; i0 < parts; i0 += 4*wpp)
        {
            // four at a time: the loads' latency is what this costs
            float2 ts[4];
            float4 o[4];
#pragma unroll
            for(int u = 0; u < 4; ++u)
            {
                const int i = i0 + u*wpp;
                const size_t p = 2*(size_t)(first + i) + (i == 0 ? 1 : 0);
                const bool on = i < parts;
                ts[u] = on ? a.part_sums[(p*MT + m)*8 + head] : make_float2(-CUDART_INF_F, 0.0f);
                o[u] = on ? *reinterpret_cast<const float4 *>(a.part_o + (p*MT + m)*8*DP + off)
                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            join_add(s, ts, o);
        }
    }
    if(wpp > 1)
    {
        if((lane & 15) == 0)
        {
            sums_s[warp][lane >> 4] = make_float2(s.top, s.sum);
        }
        o_s[warp][lane] = s.o;
        __syncthreads();
        if(warp % wpp != 0)
        {
            return;
        }
        for(int w0 = 1; w0 < wpp; w0 += 4)
        {
            float2 ts[4];
            float4 o[4];
#pragma unroll
            for(int u = 0; u < 4; ++u)
            {
                const bool on = w0 + u < wpp;
                const int w = on ? warp + w0 + u : warp;
                ts[u] = on ? sums_s[w][lane >> 4] : make_float2(-CUDART_INF_F, 0.0f);
                o[u] = on ? o_s[w][lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            join_add(s, ts, o);
        }
    }
    if(none)
    {
        return;
    }
    const size_t qh = ((size_t)kvh*a.group + g)*a.batch + b;
    const float inv = s.sum == 0.0f ? 0.0f : 1.0f/s.sum;
    const float v[4] = {s.o.x, s.o.y, s.o.z, s.o.w};
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        if(col + i < a.head)
        {
            ((T *)a.out)[qh*a.head + col + i] = from_f<T>(v[i]*inv);
        }
    }
    if(a.lse_out && col == 0)
    {
        a.lse_out[qh] = s.sum == 0.0f ? -CUDART_INF_F
                : ((s.top == -CUDART_INF_F ? 0.0f : s.top) + log2f(s.sum))*PD_LN2;
    }
}

// Tensor-core kernel: rows of a multiple of 16 bytes on 16-byte boundaries, pages of a
// multiple of 16 positions, tiles and prefix sums that fit their integers and buffers.
struct PagedDecodePlan
{
    bool fast;
    int dp, mt, grid, wpw, whole;        // fast
    int nsplit, chunk;                   // generic
    size_t bytes;
};

static PagedDecodePlan paged_decode_plan(int64_t head, int64_t page_size, int64_t max_blocks,
        int64_t batch, int64_t group, int64_t kv_heads, int64_t num_selected, int page_format,
        int64_t num_pages = 1)
{
    PagedDecodePlan p = {};
    const int64_t listed = num_selected > 0 ? num_selected : max_blocks;
    const int64_t heads = batch*group*kv_heads;
    const bool e4m3 = page_format == NNTILE_B200_PAGES_E4M3;
    p.dp = head <= 64 ? 64 : head <= 128 ? 128 : 256;
    // two tiles of heads a pass halve the reads of groups above 8; the accumulators of 256
    // columns leave no registers for it
    p.mt = group > 8 && p.dp < 256 ? 2 : 1;
    const int64_t htiles = (group + 8*p.mt - 1)/(8*p.mt);
    const int64_t unit_tiles = listed*(page_size/PD_TILE);
    const int64_t units = batch*kv_heads*htiles;
    p.fast = page_size % PD_TILE == 0 && head % (e4m3 ? 16 : 8) == 0 && batch < 4096
            && unit_tiles*units < (int64_t)1 << 30 && units < (int64_t)1 << 24
            && num_pages > 0 && num_pages*kv_heads*page_size < (int64_t)1 << 31;
    if(p.fast)
    {
        const int warps = paged_warps(e4m3, p.dp);
        const int64_t total = unit_tiles*units;
        // Workers are warps when there are units enough for most of a warp's share to be of
        // one or two of them; with fewer units the warps of a block work together, which
        // makes a part of a unit eight times as long and the parts to join eight times fewer.
        p.wpw = units >= 2*PD_SMS ? 1 : warps;
        // Whole units, nothing to join: short ones always; longer ones when they about fill
        // the SMs once, where a block streams a unit in the time that splitting and joining
        // add.  Measured (bf16, head 128, group 4, whole against split): 512 positions 9.7
        // against 12.6 us at 64 units and 11.8 against 14.5 at 144, 1024 positions 13.3 against
        // 14.9 and 16.8 against 19.4; 2048 positions 20.5 against 19.4 and 27.8 against 30.5.
        // Selections are equally long for all units, so that there more of them may be whole.
        const bool fills = units >= PD_SMS/3 && units <= PD_SMS;
        const bool even = num_selected > 0 && units >= 2*PD_SMS/3;
        if(unit_tiles <= 2*warps || (fills && unit_tiles <= (even ? 20 : 8)*warps))
        {
            p.whole = 1;
            const int64_t per = warps/p.wpw;
            p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(PD_SMS, (units + per - 1)/per));
        }
        else
        {
            p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(PD_SMS, (total + warps - 1)/warps));
            p.bytes = (size_t)2*p.grid*warps*p.mt*8*(p.dp*sizeof(float) + sizeof(float2))
                    + (size_t)units*sizeof(int2);
        }
    }
    const int64_t rows = listed*page_size;
    int64_t nsplit = (PD_SMS*8 + heads - 1)/std::max<int64_t>(heads, 1);
    nsplit = std::min(nsplit, (rows + 255)/256);
    nsplit = std::max<int64_t>(1, std::min(nsplit, std::max<int64_t>(listed, 1)));
    const int64_t chunk = std::max<int64_t>(1, (listed + nsplit - 1)/nsplit);
    p.chunk = (int)chunk;
    p.nsplit = (int)std::max<int64_t>(1, (listed + chunk - 1)/chunk);
    return p;
}

static size_t paged_generic_bytes(const PagedDecodePlan &p, int64_t head, int64_t heads)
{
    return (size_t)heads*p.nsplit*(size_t)(head + 1)*sizeof(float);
}

// What a caller provides: enough for either page format and any alignment of the pages.
static size_t paged_decode_bytes(int64_t head, int64_t page_size, int64_t max_blocks,
        int64_t batch, int64_t group, int64_t kv_heads, int64_t num_selected)
{
    size_t most = 16;
    for(int format : {NNTILE_B200_PAGES_SAME, NNTILE_B200_PAGES_E4M3})
    {
        const PagedDecodePlan p = paged_decode_plan(head, page_size, max_blocks, batch, group,
                kv_heads, num_selected, format);
        most = std::max(most, std::max(p.bytes, paged_generic_bytes(p, head,
                batch*group*kv_heads)));
    }
    return most;
}

template<typename T, bool E4M3, int DP, int MT, bool EXACT>
static int launch_main(cudaStream_t s, const PagedDecodeArgs &a, const PagedDecodePlan &plan)
{
    using L = PagedTile<E4M3, DP>;
    static PerDeviceOnce once;
    int dev = -1;
    if(cudaGetDevice(&dev) != cudaSuccess || !once.ensure(dev, []
    {
        return cudaFuncSetAttribute(paged_decode_kernel<T, E4M3, DP, MT, EXACT>,
                cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM) == cudaSuccess;
    }))
    {
        return NNTILE_B200_E_LAUNCH;
    }
    return launch_chained(paged_decode_kernel<T, E4M3, DP, MT, EXACT>, dim3(plan.grid),
            L::WARPS*32, L::SMEM, s, a);
}

template<typename T, bool E4M3, int DP, int MT>
static int launch_fast(cudaStream_t s, const PagedDecodeArgs &a, const PagedDecodePlan &plan)
{
    const int st = a.head == DP ? launch_main<T, E4M3, DP, MT, true>(s, a, plan)
            : launch_main<T, E4M3, DP, MT, false>(s, a, plan);
    if(st != NNTILE_B200_OK || a.whole) return st;
    // starts while the first kernel still runs and waits for its results on the device
    const int htiles = (a.group + 8*MT - 1)/(8*MT);
    // warps a piece: about as many as it has parts by fours, were the lengths even; with
    // uneven ones a unit may have more, so never one alone when blocks are the workers.
    // Measured with 8, 16 and 32 (bf16, head 128, group 4): 64 parts 10.4, 9.9 and 10.6 us, 74
    // parts 26.8, 25.4 and 25.5, 148 parts 18.5, 18.1 and 17.7; 18 parts 10.4 and 10.8 with 8 and
    // 16.
    const int64_t units = (int64_t)a.batch*a.kv_heads*htiles;
    const int wpp = a.wpw == 1 ? 1 : plan.grid <= 3*units ? 4 : plan.grid <= 20*units ? 8
            : plan.grid <= 72*units ? 16 : 32;
    const int64_t warps = units*join_pieces(std::min(8*MT, a.group), DP)*wpp;
    const int block = std::max(wpp, 8);
    auto kernel = wpp == 32 ? paged_join_kernel<T, E4M3, DP, MT, 32>
            : wpp == 16 ? paged_join_kernel<T, E4M3, DP, MT, 16>
            : paged_join_kernel<T, E4M3, DP, MT, 8>;
    return launch_chained(kernel, dim3((unsigned)((warps + block - 1)/block)), block*32, 0, s, a,
            plan.grid*(paged_warps(E4M3, DP)/a.wpw), wpp);
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
    PagedDecodePlan plan = paged_decode_plan(head, page_size, max_blocks, batch, group, kv_heads,
            num_selected, page_format, num_pages);
    const int64_t heads = batch*group*kv_heads;
    const uintptr_t rows16 = (uintptr_t)k_pages | (uintptr_t)v_pages
            | (e4m3 ? (uintptr_t)k_scales | (uintptr_t)v_scales : 0);
    plan.fast = plan.fast && (rows16 & 15) == 0 && ((uintptr_t)q & 3) == 0;
    if(!plan.fast && heads*plan.nsplit > INT32_MAX) return NNTILE_B200_E_SHAPE;
    if(workspace_bytes < paged_decode_bytes(head, page_size, max_blocks, batch, group, kv_heads,
            num_selected))
    {
        return NNTILE_B200_E_SCRATCH;
    }
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
    a.part_lse = a.part_o + (size_t)heads*plan.nsplit*(size_t)head;      // generic kernel
    a.part_sums = reinterpret_cast<float2 *>(a.part_o + (plan.fast
            ? (size_t)2*plan.grid*paged_warps(e4m3, plan.dp)*plan.mt*8*plan.dp : 0));
    a.spans = reinterpret_cast<int2 *>(a.part_sums + (plan.fast
            ? (size_t)2*plan.grid*paged_warps(e4m3, plan.dp)*plan.mt*8 : 0));
    a.wpw = plan.wpw;
    a.whole = plan.whole;
    a.status = status;
    a.nsplit = plan.nsplit;
    a.chunk = plan.chunk;
    cudaStream_t s = as_stream(stream);
    if(plan.fast)
    {
#define NB200_PD(E, P, M) launch_fast<T, E, P, M>(s, a, plan)
#define NB200_PD_P(E) (plan.dp == 64 ? (plan.mt == 1 ? NB200_PD(E, 64, 1) : NB200_PD(E, 64, 2)) \
        : plan.dp == 128 ? (plan.mt == 1 ? NB200_PD(E, 128, 1) : NB200_PD(E, 128, 2)) \
        : NB200_PD(E, 256, 1))
        return e4m3 ? NB200_PD_P(true) : NB200_PD_P(false);
#undef NB200_PD_P
#undef NB200_PD
    }
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

// Compiled twice, once per row type (-DNB200_FP16), to keep the build short.
#ifndef NB200_FP16
extern "C" size_t nntile_b200_paged_decode_sdpa_workspace_bytes(int64_t head, int64_t page_size,
        int64_t max_blocks, int64_t batch, int64_t group, int64_t kv_heads, int64_t num_selected)
{
    if(check_paged(head, page_size, 0, max_blocks, batch, kv_heads, NNTILE_B200_PAGES_SAME)
            != NNTILE_B200_OK || group < 0 || group > 1 << 16 || num_selected < 0
            || num_selected > INT32_MAX/page_size)
    {
        return 0;
    }
    return paged_decode_bytes(head, page_size, max_blocks, batch, group, kv_heads, num_selected);
}

#endif // NB200_FP16

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

#ifdef NB200_FP16
NB200_PAGED_DECODE_ENTRY(fp16, __half)
#else
NB200_PAGED_DECODE_ENTRY(bf16, bf16)
#endif
