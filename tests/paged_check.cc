// Host check of nntile_b200/csrc/paged_check.hh: what the paged-cache kernels do with odd
// lengths, page numbers and selections that they find in device memory.
#include <climits>
#include <cstdio>
#include <initializer_list>

#include "../nntile_b200/csrc/paged_check.hh"

using namespace nb200;

#define CHECK(x) do { if(!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while(0)

int main()
{
    const int odd[] = {INT_MIN, INT_MIN + 1, -2, -1, 0, 1, 2, 15, 16, 17, 1000, INT_MAX - 1, INT_MAX};
    for(int cap : {0, 1, 16, 1000, INT_MAX})
    {
        for(int v : odd)
        {
            bool bad = false;
            const int len = held_length(v, cap, bad);
            CHECK(len >= 0 && len <= cap);
            CHECK(bad == (v < 0 || v > cap));
            CHECK(bad || len == v);
            CHECK(page_in_pool(v, cap) == (v >= 0 && v < cap));
            for(int start : {0, cap/2, cap})
            {
                for(int n : {0, 1, 17, 1 << 20})
                {
                    bad = false;
                    const int count = held_count(v, n, start, cap, bad);
                    CHECK(count >= 0 && count <= n && (int64_t)start + count <= cap);
                    CHECK(bad == (v < 0 || v > n || v > cap - start));
                }
            }
            bad = false;
            const int blk = held_block(v, cap/2, cap, bad);
            CHECK(blk == -1 || (blk == v && blk >= 0 && blk < cap/2));
            CHECK(bad == (v >= cap));
        }
    }
    // every row of a run lands in exactly one of the blocks a launch visits
    for(int page : {1, 2, 5, 16, 64})
    {
        for(int start = 0; start < 3*page; ++start)
        {
            for(int count = 0; count <= 4*page + 1; ++count)
            {
                int rows = 0, next = start;
                for(int j = 0; j < most_touched(count, page); ++j)
                {
                    int first, last;
                    const int block = start/page + j;
                    rows_in_block(start, count, block, page, first, last);
                    CHECK(first >= 0 && last <= page);
                    if(first < last)
                    {
                        CHECK(block*page + first == next);
                        next += last - first;
                        rows += last - first;
                    }
                }
                CHECK(rows == count);
            }
        }
        CHECK(blocks_of(0, page) == 0 && blocks_of(1, page) == 1 && blocks_of(page, page) == 1);
        CHECK(blocks_of(page + 1, page) == 2 || page == 0);
    }
    CHECK(blocks_of(INT_MAX, 16) == 134217728);
    int first, last;
    rows_in_block(INT_MAX - 1, 1, INT_MAX/16, 16, first, last);
    CHECK(first == 14 && last == 15);
    rows_in_block(0, INT_MAX, INT_MAX/65536 + 1, 65536, first, last);
    CHECK(first >= last);
    return 0;
}
