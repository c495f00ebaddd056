// paged.h -- the paged KV cache shared by the append and attention kernels.
//
// A cache is n_pages pages of page_size rows each, a row being one position
// in the ring caches' layout ([n_kv_heads][head_dim] values of the cache's
// format), so that a ring cache read in page_size steps is a paged one.  A
// place is page * page_size + offset.  Page tables, lengths and slots come from
// device memory: whatever they hold, a kernel touches no place outside the
// cache; it leaves such a place out and says so in the context's
// page_faults, which mrml_hip_sync turns into an error.
#pragma once

#include "device.h"
#include "internal.h"
#include "page_map.h"

namespace mrml {

__device__ __forceinline__ void page_fault(uint32_t *faults)
{
    __hip_atomic_store(faults, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// Bytes of one head's row in a cache format (0 f16, 1 Q8_0, 2 Q4_0).
__host__ __device__ constexpr int kv_row_bytes(int fmt, int head_dim)
{
    return fmt == 0 ? head_dim * 2 : head_dim / 32 * (fmt == 1 ? 34 : 18);
}

struct BlockTablesArgs {
    const int32_t *lens, *want;
    int32_t *table;
    int32_t *free_pages;
    const int32_t *n_free;
    int32_t *lens_out, *n_free_out, *row_start, *slots, *pos, *status;
    int n_seqs, table_stride, max_rows, pos0;
    PageMap map;
    uint32_t *faults;
};

struct PagedAttn {
    const float *q;
    const uint8_t *k, *v;
    float *out;
    const int32_t *prefix, *table, *lens, *row_start;
    uint32_t *faults;
    PageMap map;
    int q_stride, prefix_len, table_stride, n_seqs, max_rows;
    int n_heads, n_kv_heads, head_dim, group;
    uint32_t group_magic;  // ceil(2^32 / group), 0 for 1
    int longest;           // positions of a table row
    int window;  // 0: none
    int k_fmt, v_fmt;
    float scale;
};

// Whether a call's units of work can be counted in 32 bits.
bool paged_attn_countable(const PagedAttn &a);
size_t paged_attn_scratch_bytes(const PagedAttn &a);
int launch_paged_attn(mrml_hip_ctx *ctx, const PagedAttn &a, void *scratch);

}  // namespace mrml
