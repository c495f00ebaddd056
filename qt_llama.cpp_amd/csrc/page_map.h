// page_map.h -- where a position lies in a paged cache (host and device).
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define MRML_PM_HD __host__ __device__ __forceinline__
#else
#define MRML_PM_HD static inline
#endif

namespace mrml {

constexpr int kMaxPageSize = 2048;
constexpr int kMaxTablePositions = 1 << 21;  // table_stride * page_size, prefix_len

// pos / page_size for pos < 2^21 by one multiplication: with magic =
// floor(2^32 / page_size) + 1 the quotient is exact while pos * page_size <
// 2^32, which the two limits above keep (page_size 1 has no 32-bit magic: 0).
struct PageMap {
    int n_pages, page_size;
    uint32_t magic;
};

inline PageMap page_map(int n_pages, int page_size)
{
    return PageMap{n_pages, page_size, page_size > 1 ? (uint32_t)((1ull << 32) / (uint32_t)page_size) + 1u : 0u};
}

MRML_PM_HD int page_of(const PageMap &m, int pos)
{
    return m.magic ? (int)(((uint64_t)(uint32_t)pos * m.magic) >> 32) : pos;
}

// The place of position pos in the cache given the id of its page; -1 for an
// id outside the cache.
MRML_PM_HD int place_of(const PageMap &m, int pos, int page, int id)
{
    return id >= 0 && id < m.n_pages ? id * m.page_size + (pos - page * m.page_size) : -1;
}

}  // namespace mrml
