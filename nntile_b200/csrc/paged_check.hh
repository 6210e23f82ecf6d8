// Index arithmetic of the paged-cache kernels that reads values a caller left in device
// memory: which of them may be used, and which positions a call touches.  Plain C++ (no
// CUDA headers needed), so that a host-only test can drive it over every odd value.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define NB200_HD __host__ __device__ __forceinline__
#else
#define NB200_HD inline
#endif

namespace nb200 {

// Filled positions a table of `capacity` positions can hold; `bad` is set when the stored
// length is not one of them.
NB200_HD int held_length(int length, int capacity, bool &bad)
{
    if(length < 0 || length > capacity)
    {
        bad = true;
        return length < 0 ? 0 : capacity;
    }
    return length;
}

NB200_HD bool page_in_pool(int page, int num_pages)
{
    return (unsigned)page < (unsigned)num_pages;
}

// Blocks that hold `length` positions.
NB200_HD int blocks_of(int length, int page_size)
{
    return length/page_size + (length % page_size != 0 ? 1 : 0);
}

// Rows an append may write for one sequence: the stored count held to [0, new_seq] and to
// the room behind `start`.
NB200_HD int held_count(int count, int new_seq, int start, int capacity, bool &bad)
{
    if(count < 0 || count > new_seq)
    {
        bad = true;
        count = count < 0 ? 0 : new_seq;
    }
    if(count > capacity - start)
    {
        bad = true;
        count = capacity - start;
    }
    return count;
}

// Positions [first, last) inside block `block` that a run of `count` rows from `start` on
// writes; empty (first >= last) when it touches none of them.
NB200_HD void rows_in_block(int start, int count, int block, int page_size, int &first, int &last)
{
    const int64_t origin = (int64_t)block*page_size;
    const int64_t lo = start - origin, hi = (int64_t)start + count - origin;
    first = lo > 0 ? (int)(lo < page_size ? lo : page_size) : 0;
    last = hi > 0 ? (int)(hi < page_size ? hi : page_size) : 0;
}

// Most blocks that `new_seq` consecutive rows can touch: a run that starts on the last row
// of a page.
NB200_HD int64_t most_touched(int64_t new_seq, int64_t page_size)
{
    return new_seq > 0 ? (new_seq + page_size - 2)/page_size + 1 : 0;
}

// A selected block as a kernel may use it: -1 when it adds nothing (a negative entry, or
// one behind the sequence's blocks); `bad` when the table could not hold it.
NB200_HD int held_block(int block, int blocks, int max_blocks, bool &bad)
{
    if(block >= max_blocks)
    {
        bad = true;
        return -1;
    }
    return block >= 0 && block < blocks ? block : -1;
}

// End of the list positions that split `split` of `chunk` positions each takes.
NB200_HD int split_end(int listed, int split, int chunk)
{
    const int64_t end = ((int64_t)split + 1)*chunk;
    return end < listed ? (int)end : listed;
}

} // namespace nb200
