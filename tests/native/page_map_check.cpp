// Checks page_map.h on the host: the quotient of every page size at the
// positions around each page's ends, and places for ids inside and outside.
#include <cstdint>
#include <cstdio>

#include "../../qt_llama.cpp_amd/csrc/page_map.h"

using namespace mrml;

int main()
{
    long bad = 0;
    for (int ps = 1; ps <= kMaxPageSize; ++ps) {
        const PageMap m = page_map(5, ps);
        for (int first = 0; first <= kMaxTablePositions; first += ps)
            for (int pos = first > 0 ? first - 1 : 0; pos <= first + 1 && pos <= kMaxTablePositions; ++pos)
                bad += page_of(m, pos) != pos / ps;
        for (int id = -3; id < 9; ++id)
            for (int pos = 0; pos < 3 * ps; pos += ps > 64 ? 37 : 1) {
                const int want = id >= 0 && id < 5 ? id * ps + pos % ps : -1;
                bad += place_of(m, pos, page_of(m, pos), id) != want;
            }
        bad += place_of(m, 0, 0, INT32_MIN) != -1 || place_of(m, 0, 0, INT32_MAX) != -1;
    }
    const PageMap large = page_map(INT32_MAX / 2048, 2048);  // the largest cache: its last place
    const int last = large.n_pages - 1, place = place_of(large, 2047, 0, last);
    bad += place != (int)((int64_t)last * 2048 + 2047) || place < 0;
    std::printf("%ld\n", bad);
    return bad != 0;
}
