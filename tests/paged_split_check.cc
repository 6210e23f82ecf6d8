// Host check of nntile_b200/csrc/paged_check.hh: splits of a list, however long, take every
// position of it once.
#include <climits>
#include <cstdio>
#include <initializer_list>

#include "../nntile_b200/csrc/paged_check.hh"

using namespace nb200;

#define CHECK(x) do { if(!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while(0)

int main()
{
    for(int most : {1, 2, 255, 256, 257, 100003, INT_MAX/2, INT_MAX - 95, INT_MAX - 1, INT_MAX})
    {
        for(int64_t wanted : {1, 2, 3, 148, 1184, 1185})
        {
            // as the launch divides a table of `most` blocks
            const int64_t chunk = (most + wanted - 1)/wanted;
            const int nsplit = (int)((most + chunk - 1)/chunk);
            for(int listed : {0, 1, most/2, most - 1, most})
            {
                int64_t next = 0;
                for(int split = 0; split < nsplit; ++split)
                {
                    const int64_t begin = (int64_t)split*chunk;
                    const int end = split_end(listed, split, (int)chunk);
                    CHECK(begin <= INT_MAX && end <= listed);
                    if(begin < end)
                    {
                        CHECK(begin == next);
                        next = end;
                    }
                }
                CHECK(next == listed);
            }
        }
    }
    return 0;
}
