// Writing a paged key/value cache and reading it back.
//
// Both kernels move bytes; the bound is HBM bandwidth for prompts and the chain of memory
// latencies (length, page and row, old bounds) for single tokens.  What they spend beside the
// copies is instructions, so those are what is kept few: rows are fetched four ahead, where a
// row lies is worked out once per row and not in each of its lanes, maxima and bounds go
// through packed or 16-byte accesses.
//
// Measured on one B200 (copy bandwidth 6 553 GB/s): append of one row for each of 64 sequences,
// 8 heads of 128, with bounds: 4.4 us (e4m3: 3.6); of prompts of up to 4096 rows for 4 sequences,
// fp16 with bounds: 19.8 us, 5.4 TB/s of read and written rows; 4096 bf16 rows for 4 sequences
// into e4m3 pages with bounds: 29 us, 3.4 TB/s; up to 1023 bf16 rows for 8 sequences into
// e4m3 pages and all of their up to 6000 rows read back: 39 us, 5.2 TB/s; read-back of 16 x
// up to 8192 bf16 rows: 111 us, 6.5 TB/s.
#include <algorithm>

#include "paged.cuh"

namespace nb200 {

constexpr int ROW_THREADS = 128;
constexpr int ROWS_AHEAD = 4;
constexpr int PART_ROWS = 32;
constexpr int GATHER_ROWS = 64;

// Elements a lane owns of a row.  VEC: eight neighbouring ones, one 16-byte access, LPR
// lanes a row (LPR = 8, 16, 32 for heads up to 64, 128, 256).  Otherwise (a head that is
// not a multiple of 8, or pointers off a 16-byte boundary) every 32nd one, a warp a row.
template<bool VEC, int LPR>
__device__ __forceinline__ int element(int lane, int i)
{
    return VEC ? 8*(lane & (LPR - 1)) + i : lane + 32*i;
}

// The eight elements as they lie in memory: fetched for several rows before the first is
// used, so that a thread has that many loads in flight.
template<typename T, bool VEC, int LPR>
__device__ __forceinline__ uint4 fetch_row(const T *row, int head, int lane, bool live)
{
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if(VEC)
    {
        const int h = element<VEC, LPR>(lane, 0);
        return live && h < head ? *reinterpret_cast<const uint4 *>(row + h)
                : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for(int i = 0; i < 8; ++i)
    {
        const int h = element<VEC, LPR>(lane, i);
        unsigned short v = 0;
        if(live && h < head)
        {
            v = reinterpret_cast<const unsigned short *>(row)[h];
        }
        w[i >> 1] |= (uint32_t)v << 16*(i & 1);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template<typename T>
__device__ __forceinline__ void widen(const uint4 &v, float (&x)[8])
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const float2 f = unpack2<T>(w[i]);
        x[2*i] = f.x;
        x[2*i + 1] = f.y;
    }
}

template<typename T, bool VEC, int LPR>
__device__ __forceinline__ void store_row(T *row, int head, int lane, const uint4 &v)
{
    if(VEC)
    {
        const int h = element<VEC, LPR>(lane, 0);
        if(h < head)
        {
            *reinterpret_cast<uint4 *>(row + h) = v;
        }
    }
    else
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int h = element<VEC, LPR>(lane, i);
            if(h < head)
            {
                reinterpret_cast<unsigned short *>(row)[h] = (unsigned short)(w[i >> 1]
                        >> 16*(i & 1));
            }
        }
    }
}

template<typename T>
__device__ __forceinline__ uint4 narrow(const float (&x)[8])
{
    return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
            pack2<T>(x[6], x[7]));
}

template<bool VEC, int LPR>
__device__ __forceinline__ void store_codes(uint8_t *row, int head, int lane,
        const uint32_t (&c)[4])
{
    if(VEC)
    {
        const int h = element<VEC, LPR>(lane, 0);
        if(h < head)
        {
            *reinterpret_cast<uint2 *>(row + h) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int h = element<VEC, LPR>(lane, i);
            if(h < head)
            {
                row[h] = (uint8_t)(c[i >> 1] >> 8*(i & 1));
            }
        }
    }
}

template<bool VEC, int LPR>
__device__ __forceinline__ uint2 fetch_codes(const uint8_t *row, int head, int lane, bool live)
{
    if(VEC)
    {
        const int h = element<VEC, LPR>(lane, 0);
        return live && h < head ? *reinterpret_cast<const uint2 *>(row + h)
                : make_uint2(0u, 0u);
    }
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for(int i = 0; i < 8; ++i)
    {
        const int h = element<VEC, LPR>(lane, i);
        if(live && h < head)
        {
            w[i >> 2] |= (uint32_t)row[h] << 8*(i & 3);
        }
    }
    return make_uint2(w[0], w[1]);
}

// Quantise the eight elements a lane owns (its row shared by the LPR lanes around it):
// returns the exponent byte, leaves the codes in `c`.  The largest magnitude is found on
// packed pairs; only a row that holds an infinity goes through the elements one by one.
// The format has no infinity: what is not finite is kept as NaN.
template<typename T, int LPR>
__device__ __forceinline__ uint32_t quantise_row(const uint4 &raw, uint32_t (&c)[4])
{
    constexpr uint32_t ABS = 0x7FFF7FFFu;
    uint32_t top = max2<T>(max2<T>(raw.x & ABS, raw.y & ABS), max2<T>(raw.z & ABS, raw.w & ABS));
#pragma unroll
    for(int o = LPR/2; o > 0; o >>= 1)
    {
        top = max2<T>(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const float2 two = unpack2<T>(top);
    float amax = fmaxf(fmaxf(two.x, two.y), 0.0f);           // all NaN: 0
    float x[8];
    widen<T>(raw, x);
    if(__any_sync(0xffffffffu, amax == CUDART_INF_F))
    {
        amax = 0.0f;
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const float a = fabsf(x[i]);
            amax = a < CUDART_INF_F ? fmaxf(amax, a) : amax;
            x[i] = a < CUDART_INF_F ? x[i] : CUDART_NAN_F;
        }
#pragma unroll
        for(int o = LPR/2; o > 0; o >>= 1)
        {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        }
    }
    const uint32_t byte = scale_byte(amax);
    const float inv = inverse_scale(byte);
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        c[i] = f2_to_e4m3x2(x[2*i]*inv, x[2*i + 1]*inv);
    }
    return byte;
}

// A CTA writes up to PART_ROWS new rows of one (sequence, kv head, touched block): of K for an
// even blockIdx.y, of V for an odd one.  With bounds the first K part takes all rows of the
// block instead: because no other CTA writes this (page, kv head), it needs no atomics.  Four
// rows a thread are fetched before the first is stored, the first ones before the page is
// known: a step of one token is a chain of memory latencies and nothing else.
// A block's bounds are those of its stored (for 8-bit pages: quantised) keys, rounded to T;
// rows that were in the page before are merged in unless the block starts with this call.
template<typename T, bool E4M3, bool VEC, int LPR, bool BOUNDS>
__global__ void __launch_bounds__(ROW_THREADS)
paged_append_kernel(int head, int page_size, int num_pages, int max_blocks, int batch,
        int kv_heads, int new_seq, int touched, int page_shift,
        const int32_t *lengths,
        const int32_t *new_lens, const int32_t *block_table,
        const T *k, const T *v, void *k_pages,
        void *v_pages, uint8_t *k_scales,
        uint8_t *v_scales, T *bounds, uint32_t *status)
{
    constexpr int SLOTS = ROW_THREADS/LPR;       // rows in flight per CTA
    const int lane = threadIdx.x & 31;
    const int slot = threadIdx.x/LPR;
    const int unit = blockIdx.x/touched, j = blockIdx.x - unit*touched;
    const int b = unit % batch, kvh = unit/batch;
    const int capacity = max_blocks*page_size;
    chain_wait();
    const int start = checked_length(lengths, b, capacity, status);
    bool bad = false;
    const int count = held_count(new_lens ? new_lens[b] : new_seq, new_seq, start, capacity, bad);
    if(bad)
    {
        report(status, NNTILE_B200_PAGED_BAD_LENGTH);
    }
    const int block = (page_shift >= 0 ? start >> page_shift : start/page_size) + j;
    int first, last;
    rows_in_block(start, count, block, page_size, first, last);
    const bool is_k = (blockIdx.y & 1) == 0;
    const bool bounded = BOUNDS && is_k && bounds != nullptr;
    const int part = blockIdx.y >> 1;
    if(!bounded)
    {
        first += part*PART_ROWS;
        last = min(last, first + PART_ROWS);
    }
    if(first >= last || (bounded && part > 0))
    {
        return;
    }
    const int rows = last - first;
    const T *src = (is_k ? k : v) + ((size_t)unit*new_seq + ((size_t)block*page_size + first
            - start))*head;
    uint4 raw[ROWS_AHEAD];
#pragma unroll
    for(int u = 0; u < ROWS_AHEAD; ++u)
    {
        const int row = u*SLOTS + slot;
        raw[u] = fetch_row<T, VEC, LPR>(src + (size_t)row*head, head, lane, row < rows);
    }
    const int page = checked_page(block_table + (size_t)b*max_blocks, block, num_pages, status);
    if(page < 0)
    {
        return;
    }
    const size_t dst0 = ((size_t)page*kv_heads + kvh)*page_size + first;
    // what the bounds were: head <= 256 elements on 128 threads
    T *low_g = bounds + ((size_t)page*kv_heads + kvh)*2*head, *high_g = low_g + head;
    float low_was[2], high_was[2];
#pragma unroll
    for(int i = 0; i < 2; ++i)
    {
        const int h = threadIdx.x + i*ROW_THREADS;
        const bool old = bounded && first > 0 && h < head;
        low_was[i] = old ? to_f(low_g[h]) : CUDART_INF_F;
        high_was[i] = old ? to_f(high_g[h]) : -CUDART_INF_F;
    }
    float low[8], high[8];
#pragma unroll
    for(int i = 0; i < 8; ++i)
    {
        low[i] = CUDART_INF_F;
        high[i] = -CUDART_INF_F;
    }
    // warps stay converged: the quantiser shuffles within a row's lanes
    void *pages = is_k ? k_pages : v_pages;
    uint8_t *scales = is_k ? k_scales : v_scales;
    for(int r0 = 0; r0 < rows; r0 += ROWS_AHEAD*SLOTS)
    {
#pragma unroll
        for(int u = 0; u < ROWS_AHEAD; ++u)
        {
            const int row = r0 + u*SLOTS + slot;
            const bool live = row < rows;
            const size_t dst = dst0 + row;
            float x[8];
            if(E4M3)
            {
                if(r0 + u*SLOTS >= rows)
                {
                    break;                       // the whole CTA
                }
                uint32_t c[4];
                const uint32_t byte = quantise_row<T, LPR>(raw[u], c);
                if(bounded)
                {
                    const float scale = scale_value(byte);
#pragma unroll
                    for(int i = 0; i < 4; ++i)
                    {
                        const float2 back = e4m3x2_to_f2(c[i]);
                        x[2*i] = back.x*scale;
                        x[2*i + 1] = back.y*scale;
                    }
                }
                if(live)
                {
                    store_codes<VEC, LPR>((uint8_t *)pages + dst*head, head, lane, c);
                    if((lane & (LPR - 1)) == 0)
                    {
                        scales[dst] = (uint8_t)byte;
                    }
                }
            }
            else if(live)
            {
                store_row<T, VEC, LPR>((T *)pages + dst*head, head, lane, raw[u]);
            }
            if(bounded && live)
            {
                if(!E4M3)
                {
                    widen<T>(raw[u], x);
                }
#pragma unroll
                for(int i = 0; i < 8; ++i)
                {
                    low[i] = min_nan(low[i], x[i]);
                    high[i] = max_nan(high[i], x[i]);
                }
            }
        }
        if(r0 + ROWS_AHEAD*SLOTS < rows)
        {
#pragma unroll
            for(int u = 0; u < ROWS_AHEAD; ++u)
            {
                const int row = r0 + (u + ROWS_AHEAD)*SLOTS + slot;
                raw[u] = fetch_row<T, VEC, LPR>(src + (size_t)row*head, head, lane, row < rows);
            }
        }
    }
    if(!bounded)
    {
        return;
    }
    __shared__ __align__(16) float low_s[SLOTS][8*LPR], high_s[SLOTS][8*LPR];
    if(VEC)
    {
        const int h = element<VEC, LPR>(lane, 0);
#pragma unroll
        for(int i = 0; i < 8; i += 4)
        {
            *reinterpret_cast<float4 *>(&low_s[slot][h + i]) = make_float4(low[i], low[i + 1],
                    low[i + 2], low[i + 3]);
            *reinterpret_cast<float4 *>(&high_s[slot][h + i]) = make_float4(high[i],
                    high[i + 1], high[i + 2], high[i + 3]);
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            low_s[slot][element<VEC, LPR>(lane, i)] = low[i];
            high_s[slot][element<VEC, LPR>(lane, i)] = high[i];
        }
    }
    __syncthreads();
#pragma unroll
    for(int i = 0; i < 2; ++i)
    {
        const int h = threadIdx.x + i*ROW_THREADS;
        if(h < head)
        {
            float a = low_was[i], z = high_was[i];
#pragma unroll
            for(int s = 0; s < SLOTS; ++s)
            {
                a = min_nan(a, low_s[s][h]);
                z = max_nan(z, high_s[s][h]);
            }
            low_g[h] = from_f<T>(a);
            high_g[h] = from_f<T>(z);
        }
    }
}

// Rows [0, lengths[b]) of every sequence, K and V, out of the pages; rows behind are left
// as they are.  blockIdx.y: 0 = K, 1 = V.
template<typename T, bool E4M3, bool VEC, int LPR>
__global__ void __launch_bounds__(ROW_THREADS)
paged_gather_kernel(int head, int page_size, int num_pages, int max_blocks, int batch,
        int kv_heads, int max_seq, int chunks, int page_shift,
        const int32_t *lengths, const int32_t *block_table,
        const void *k_pages, const void *v_pages,
        const uint8_t *k_scales, const uint8_t *v_scales,
        T *k, T *v, uint32_t *status)
{
    constexpr int SLOTS = ROW_THREADS/LPR;
    const int lane = threadIdx.x & 31;
    const int slot = threadIdx.x/LPR;
    const int unit = blockIdx.x/chunks, chunk = blockIdx.x - unit*chunks;
    const int b = unit % batch, kvh = unit/batch;
    chain_wait();
    int len = checked_length(lengths, b, max_blocks*page_size, status);
    if(len > max_seq)
    {
        report(status, NNTILE_B200_PAGED_BAD_LENGTH);
        len = max_seq;
    }
    const bool is_k = blockIdx.y == 0;
    const void *pages = is_k ? k_pages : v_pages;
    const uint8_t *scales = is_k ? k_scales : v_scales;
    T *out = (is_k ? k : v) + (size_t)unit*max_seq*head;
    const int64_t begin = (int64_t)chunk*GATHER_ROWS;
    const int rows = (int)min((int64_t)GATHER_ROWS, len - begin);
    if(rows <= 0)
    {
        return;
    }
    // where the rows are, once per row: the lanes that share a row would all work it out
    __shared__ int64_t from_s[GATHER_ROWS];
    if(threadIdx.x < rows)
    {
        const int r = (int)begin + threadIdx.x;
        const int block = page_shift >= 0 ? r >> page_shift : r/page_size;
        const int page = checked_page(block_table + (size_t)b*max_blocks, block, num_pages, status);
        from_s[threadIdx.x] = page < 0 ? -1
                : ((int64_t)page*kv_heads + kvh)*page_size + (r - block*page_size);
    }
    __syncthreads();
    // four rows at a time are fetched together
    for(int r0 = 0; r0 < rows; r0 += ROWS_AHEAD*SLOTS)
    {
        size_t src[ROWS_AHEAD];
        bool live[ROWS_AHEAD];
#pragma unroll
        for(int u = 0; u < ROWS_AHEAD; ++u)
        {
            const int r = r0 + u*SLOTS + slot;
            const int64_t from = r < rows ? from_s[r] : -1;
            live[u] = from >= 0;
            src[u] = (size_t)max(from, (int64_t)0);
        }
        uint4 raw[ROWS_AHEAD];
        uint32_t byte[ROWS_AHEAD];
#pragma unroll
        for(int u = 0; u < ROWS_AHEAD; ++u)
        {
            if(E4M3)
            {
                const uint2 c = fetch_codes<VEC, LPR>((const uint8_t *)pages + src[u]*head, head,
                        lane, live[u]);
                raw[u] = make_uint4(c.x, c.y, 0u, 0u);
                byte[u] = live[u] ? scales[src[u]] : 0u;
            }
            else
            {
                raw[u] = fetch_row<T, VEC, LPR>((const T *)pages + src[u]*head, head, lane,
                        live[u]);
            }
        }
#pragma unroll
        for(int u = 0; u < ROWS_AHEAD; ++u)
        {
            if(E4M3)
            {
                const float scale = scale_value(byte[u]);
                float x[8];
#pragma unroll
                for(int i = 0; i < 4; ++i)
                {
                    const uint32_t two = (i < 2 ? raw[u].x : raw[u].y) >> 16*(i & 1) & 0xFFFFu;
                    const float2 f = e4m3x2_to_f2(two);
                    x[2*i] = f.x*scale;
                    x[2*i + 1] = f.y*scale;
                }
                raw[u] = narrow<T>(x);
            }
            if(live[u])
            {
                store_row<T, VEC, LPR>(out + (size_t)(begin + r0 + u*SLOTS + slot)*head, head, lane,
                        raw[u]);
            }
        }
    }
}

// 16-byte accesses need rows of a multiple of 8 elements on 16-byte boundaries (8 bytes for
// codes); everything else goes element by element.
static bool vector_rows(int64_t head, bool e4m3, const void *a, const void *b, const void *pa,
        const void *pb)
{
    const uintptr_t rows = (uintptr_t)a | (uintptr_t)b, pages = (uintptr_t)pa | (uintptr_t)pb;
    return head % 8 == 0 && (rows & 15) == 0 && (pages & (e4m3 ? 7 : 15)) == 0;
}

// Shift of a power of two, the usual page size; -1 for others.
static int shift_of(int64_t page_size)
{
    for(int i = 0; i <= 16; ++i)
    {
        if(page_size == (int64_t)1 << i) return i;
    }
    return -1;
}

template<typename T>
static int append_impl(nntile_b200_stream_t stream, int64_t head, int64_t page_size,
        int64_t num_pages, int64_t max_blocks, int64_t batch, int64_t kv_heads, int64_t new_seq,
        int page_format, const int32_t *lengths, const int32_t *new_lens,
        const int32_t *block_table, const void *k, const void *v, void *k_pages, void *v_pages,
        uint8_t *k_scales, uint8_t *v_scales, void *bounds, uint32_t *status)
{
    const int st = check_paged(head, page_size, num_pages, max_blocks, batch, kv_heads,
            page_format);
    if(st != NNTILE_B200_OK) return st;
    if(new_seq < 0) return NNTILE_B200_E_BADARG;
    if(new_seq > INT32_MAX/2) return NNTILE_B200_E_SHAPE;
    if(batch == 0 || kv_heads == 0 || new_seq == 0) return NNTILE_B200_OK;
    const bool e4m3 = page_format == NNTILE_B200_PAGES_E4M3;
    if(max_blocks == 0 || num_pages == 0) return NNTILE_B200_E_BADARG;      // no room at all
    if(!lengths || !block_table || !k || !v || !k_pages || !v_pages
            || (e4m3 && (!k_scales || !v_scales)))
    {
        return NNTILE_B200_E_BADARG;
    }
    if(((uintptr_t)k | (uintptr_t)v | (uintptr_t)bounds) & 1) return NNTILE_B200_E_ALIGN;
    if(!e4m3 && (((uintptr_t)k_pages | (uintptr_t)v_pages) & 1)) return NNTILE_B200_E_ALIGN;
    if(((uintptr_t)lengths | (uintptr_t)new_lens | (uintptr_t)block_table | (uintptr_t)status) & 3)
    {
        return NNTILE_B200_E_ALIGN;
    }
    const int64_t touched = std::min(most_touched(new_seq, page_size), max_blocks);
    if(touched*batch*kv_heads > INT32_MAX) return NNTILE_B200_E_SHAPE;
    // parts of a block that this call may fill
    const int64_t most = std::min(new_seq, page_size);
    const dim3 grid((unsigned)(touched*batch*kv_heads),
            (unsigned)(2*((most + PART_ROWS - 1)/PART_ROWS)));
    const bool vec = vector_rows(head, e4m3, k, v, k_pages, v_pages);
    cudaStream_t s = as_stream(stream);
#define NB200_APPEND(E, V, L) return launch_chained(bounds ? paged_append_kernel<T, E, V, L, true> \
        : paged_append_kernel<T, E, V, L, false>, grid, ROW_THREADS, 0, s, (int)head, (int)page_size, (int)num_pages, (int)max_blocks, (int)batch, (int)kv_heads, \
        (int)new_seq, (int)touched, shift_of(page_size), lengths, new_lens, block_table, (const T *)k, (const T *)v, \
        k_pages, v_pages, k_scales, v_scales, (T *)bounds, status)
#define NB200_APPEND_L(E) \
    do { \
        if(!vec) NB200_APPEND(E, false, 32); \
        else if(head <= 64) NB200_APPEND(E, true, 8); \
        else if(head <= 128) NB200_APPEND(E, true, 16); \
        else NB200_APPEND(E, true, 32); \
    } while(0)
    if(e4m3) NB200_APPEND_L(true);
    else NB200_APPEND_L(false);
#undef NB200_APPEND_L
#undef NB200_APPEND
}

template<typename T>
static int gather_impl(nntile_b200_stream_t stream, int64_t head, int64_t page_size,
        int64_t num_pages, int64_t max_blocks, int64_t batch, int64_t kv_heads, int64_t max_seq,
        int page_format, const int32_t *lengths, const int32_t *block_table,
        const void *k_pages, const void *v_pages, const uint8_t *k_scales,
        const uint8_t *v_scales, void *k, void *v, uint32_t *status)
{
    const int st = check_paged(head, page_size, num_pages, max_blocks, batch, kv_heads,
            page_format);
    if(st != NNTILE_B200_OK) return st;
    if(max_seq < 0) return NNTILE_B200_E_BADARG;
    if(max_seq > INT32_MAX) return NNTILE_B200_E_SHAPE;
    if(batch == 0 || kv_heads == 0 || max_seq == 0 || max_blocks == 0) return NNTILE_B200_OK;
    const bool e4m3 = page_format == NNTILE_B200_PAGES_E4M3;
    if(!lengths || !block_table || !k || !v || (num_pages > 0 && (!k_pages || !v_pages
            || (e4m3 && (!k_scales || !v_scales)))))
    {
        return NNTILE_B200_E_BADARG;
    }
    if(((uintptr_t)k | (uintptr_t)v) & 1) return NNTILE_B200_E_ALIGN;
    if(!e4m3 && (((uintptr_t)k_pages | (uintptr_t)v_pages) & 1)) return NNTILE_B200_E_ALIGN;
    if(((uintptr_t)lengths | (uintptr_t)block_table | (uintptr_t)status) & 3)
    {
        return NNTILE_B200_E_ALIGN;
    }
    const int64_t reach = std::min(max_seq, max_blocks*page_size);
    const int64_t chunks = (reach + GATHER_ROWS - 1)/GATHER_ROWS;
    if(chunks*batch*kv_heads > INT32_MAX) return NNTILE_B200_E_SHAPE;
    const dim3 grid((unsigned)(chunks*batch*kv_heads), 2);
    const bool vec = vector_rows(head, e4m3, k, v, k_pages, v_pages);
    cudaStream_t s = as_stream(stream);
#define NB200_GATHER(E, V, L) return launch_chained(paged_gather_kernel<T, E, V, L>, grid, \
        ROW_THREADS, 0, s, (int)head, (int)page_size, (int)num_pages, (int)max_blocks, (int)batch, (int)kv_heads, \
        (int)max_seq, (int)chunks, shift_of(page_size), lengths, block_table, k_pages, v_pages, \
        k_scales, v_scales, (T *)k, (T *)v, status)
#define NB200_GATHER_L(E) \
    do { \
        if(!vec) NB200_GATHER(E, false, 32); \
        else if(head <= 64) NB200_GATHER(E, true, 8); \
        else if(head <= 128) NB200_GATHER(E, true, 16); \
        else NB200_GATHER(E, true, 32); \
    } while(0)
    if(e4m3) NB200_GATHER_L(true);
    else NB200_GATHER_L(false);
#undef NB200_GATHER_L
#undef NB200_GATHER
}

} // namespace nb200

using namespace nb200;

#define NB200_PAGED_CACHE_ENTRY(SFX, T) \
extern "C" int nntile_b200_paged_kv_append_##SFX(nntile_b200_stream_t stream, int64_t head, \
        int64_t page_size, int64_t num_pages, int64_t max_blocks, int64_t batch, \
        int64_t kv_heads, int64_t new_seq, int page_format, const int32_t *lengths, \
        const int32_t *new_lens, const int32_t *block_table, const void *k, const void *v, \
        void *k_pages, void *v_pages, uint8_t *k_scales, uint8_t *v_scales, void *bounds, \
        uint32_t *status) \
{ \
    return append_impl<T>(stream, head, page_size, num_pages, max_blocks, batch, kv_heads, \
            new_seq, page_format, lengths, new_lens, block_table, k, v, k_pages, v_pages, \
            k_scales, v_scales, bounds, status); \
} \
extern "C" int nntile_b200_paged_kv_gather_##SFX(nntile_b200_stream_t stream, int64_t head, \
        int64_t page_size, int64_t num_pages, int64_t max_blocks, int64_t batch, \
        int64_t kv_heads, int64_t max_seq, int page_format, const int32_t *lengths, \
        const int32_t *block_table, const void *k_pages, const void *v_pages, \
        const uint8_t *k_scales, const uint8_t *v_scales, void *k, void *v, uint32_t *status) \
{ \
    return gather_impl<T>(stream, head, page_size, num_pages, max_blocks, batch, kv_heads, \
            max_seq, page_format, lengths, block_table, k_pages, v_pages, k_scales, v_scales, \
            k, v, status); \
}

NB200_PAGED_CACHE_ENTRY(bf16, bf16)
NB200_PAGED_CACHE_ENTRY(fp16, __half)
