// paged.hip -- a batch of requests over a paged KV cache: the step's page
// tables and slot maps, the K/V append to those slots, and the C ABI of the
// attention that reads them (attn_paged.hip).
//
// The reference serves one sequence from ring caches (cuda.rs:2438-2519,
// 2658-2770); these entry points carry its cache rows, RoPE and attention to
// requests that hold pages of one cache and share a prefix.

#include <algorithm>
#include <cmath>

#include "paged.h"
#include "rope.h"

namespace mrml {

namespace {

constexpr int kTablesT = 1024;     // threads of the table workgroup
constexpr int kTablesPer = 4;      // requests a thread at most
constexpr int kMaxSeqs = kTablesT * kTablesPer;
constexpr int kRowsAtOnce = 4;     // rows that a thread places side by side

__device__ __forceinline__ uint32_t add_sat(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// Inclusive sums over a wave's first LANES lanes (16 or 64), kept at 2^32 - 1 once there.
template <int LANES>
__device__ __forceinline__ uint32_t scan_lanes(uint32_t x)
{
#define SCAN_STEP(CTRL, ROWS) x = add_sat(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false))
    SCAN_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
    SCAN_STEP(0x112, 0xf);
    SCAN_STEP(0x114, 0xf);
    SCAN_STEP(0x118, 0xf);
    if (LANES == 64) {
        SCAN_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
        SCAN_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
    }
#undef SCAN_STEP
    return x;
}

// Exclusive sums of N numbers over the workgroup's threads (in thread order), the totals in t[].  Sums past 2^32
// stay at its end: they are only compared with what there is.  lds: N * 16 words of the call's own.  Every thread
// calls it.  (In 64 bits with shuffles the two calls took 5 us of 14 for 700 requests.)
template <int N>
__device__ __forceinline__ void block_exclusive(uint32_t v[N], uint32_t t[N], uint32_t *lds)
{
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t before[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t inc = scan_lanes<64>(v[k]);
        if (lane == 63) lds[k * 16 + wave] = inc;
        before[k] = __shfl_up(inc, 1, 64);
        if (lane == 0) before[k] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t all = scan_lanes<16>(lane < waves ? lds[k * 16 + lane] : 0);
        t[k] = (uint32_t)__builtin_amdgcn_readlane((int)all, 15);
        v[k] = add_sat(before[k], wave ? (uint32_t)__builtin_amdgcn_readlane((int)all, wave - 1) : 0);
    }
}

// For each x the first r of n with ends[r] > x (ends ascending), the last where there is none; the searches
// run side by side.
template <int N>
__device__ __forceinline__ void upper(const int32_t *ends, int n, const int *x, int *r)
{
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = 0;
    for (int len = n; len > 1;) {
        const int half = len >> 1;
#pragma unroll
        for (int e = 0; e < N; ++e) r[e] += ends[r[e] + half - 1] <= x[e] ? half : 0;
        len -= half;
    }
}

// The step's bookkeeping, one workgroup.  With held = ceil(len / page) and
// need = ceil((len + new) / page) - held for every request, prefix sums over
// the requests give each its rows, its new pages (taken from the top of the
// free list) and, for a finished one, the places its pages return to; the
// rows then find their request by bisection over the row ends in LDS.  It is
// bound by the latency of a few dependent round trips (lengths, free list or
// table, stores), not by its bytes, so everything runs in one launch and
// every list (rows, returned pages) is walked flat over all threads.  6 requests
// take 2.9 us; 700 with 4816 rows and 948 returned pages 9.9 us, most of it the rows'
// bisections (LDS reads).  Four rows of a thread side by side save 0.8 us of those; eight save 0.2
// more and cost 0.4 where rows are few.
__global__ __launch_bounds__(kTablesT) void block_tables_kernel(BlockTablesArgs a)
{
    extern __shared__ int32_t s_mem[];
    __shared__ uint32_t s_sum[3 * 16], s_rows[16], s_got[2 * 16];
    const int n = a.n_seqs, T = blockDim.x, tid = threadIdx.x, ps = a.map.page_size;
    int32_t *s_len = s_mem, *s_new0 = s_mem + n, *s_row = s_mem + 2 * n, *s_back = s_mem + 3 * n;
    const int per = (n + T - 1) / T, r0 = tid * per;
    const int free0 = *a.n_free, F0 = min(max(free0, 0), a.map.n_pages);
    const int longest = a.table_stride * ps;

    int len[kTablesPer], add[kTablesPer], need[kTablesPer], code[kTablesPer];
    uint32_t sum[3] = {0, 0, 0}, total[3];  // returned pages, rows, lacking pages; a request's share is below 2^22
#pragma unroll
    for (int e = 0; e < kTablesPer; ++e) {
        if (e >= per) break;
        const int r = r0 + e;
        const int l = r < n ? a.lens[r] : 0, w = r < n ? a.want[r] : 0;
        const bool bad = l < 0 || l > longest || w < -1;
        const int held = bad ? 0 : (l + ps - 1) / ps;
        const bool full = !bad && w > longest - l;
        const bool grows = !bad && !full && w > 0;
        len[e] = l;
        add[e] = grows ? w : 0;
        need[e] = grows ? (l + w + ps - 1) / ps - held : 0;
        code[e] = bad ? 4 : (full ? 2 : (w == -1 ? -1 : 0));  // -1: finished
        sum[0] += code[e] == -1 ? held : 0;
        sum[1] += add[e];
        sum[2] += need[e];
    }
    block_exclusive<3>(sum, total, s_sum);
    const uint32_t F = add_sat(F0, total[0]);
    const int F1 = (int)min(F, (uint32_t)a.map.n_pages);  // free pages once the finished requests' are back
    // more pages than there are: somebody's are counted twice, and those past the list's room are lost
    if (tid == 0 && (F0 != free0 || F > (uint32_t)a.map.n_pages)) page_fault(a.faults);
    // Served: the pages of every request so far are there, and the rows of every one so far that has its pages.  So none
    // takes a page or a row ahead of one that waits for the same, and one that waits for pages keeps no row from the others.
    bool waits[kTablesPer] = {};
    if (total[2] > (uint32_t)F1) {  // somebody waits for pages: the rows without theirs
        uint32_t asked[1] = {0}, all[1], pages = sum[2];
#pragma unroll
        for (int e = 0; e < kTablesPer; ++e) {
            if (e >= per) break;
            pages = add_sat(pages, need[e]);
            waits[e] = need[e] > 0 && pages > (uint32_t)F1;
            asked[0] += waits[e] ? 0 : add[e];
        }
        block_exclusive<1>(asked, all, s_rows);
        sum[1] = asked[0];
    }
    uint32_t got[2] = {0, 0}, all[2];
    {
        uint32_t back = sum[0], rows = sum[1], pages = sum[2];
#pragma unroll
        for (int e = 0; e < kTablesPer; ++e) {
            if (e >= per) break;
            const int r = r0 + e;
            back = add_sat(back, code[e] == -1 ? (len[e] + ps - 1) / ps : 0);
            if (r < n) {
                s_back[r] = (int32_t)min(back, (uint32_t)INT32_MAX);
                s_new0[r] = (int32_t)min(pages, (uint32_t)INT32_MAX);
                s_len[r] = len[e];
            }
            pages = add_sat(pages, need[e]);
            if (code[e] == 0 && add[e] > 0) {
                const uint32_t with = add_sat(rows, add[e]);
                code[e] = with > (uint32_t)a.max_rows ? 3 : waits[e] ? 1 : 0;
                if (!waits[e]) rows = with;
            }
            if (code[e] > 0) add[e] = need[e] = 0;
            got[0] += add[e];
            got[1] += need[e];
        }
    }
    block_exclusive<2>(got, all, s_got);
    {
        uint32_t rows = got[0];
#pragma unroll
        for (int e = 0; e < kTablesPer; ++e) {
            if (e >= per) break;
            const int r = r0 + e;
            if (r >= n) break;
            a.row_start[r] = (int32_t)rows;
            rows += add[e];
            s_row[r] = (int32_t)rows;
            a.lens_out[r] = code[e] == -1 ? 0 : len[e] + add[e];
            a.status[r] = code[e] < 0 ? 0 : code[e];
        }
    }
    const int rows = (int)all[0];
    if (tid == 0) {
        a.row_start[n] = rows;
        a.n_free_out[0] = F1 - (int)all[1];
    }
    __syncthreads();

    // finished requests' pages onto the free list
    const int returned = F1 - F0;
    for (int i = tid; i < returned; i += T) {
        int r;
        upper<1>(s_back, n, &i, &r);
        const int j = i - (r ? s_back[r - 1] : 0);
        a.free_pages[F0 + i] = a.table[(size_t)r * a.table_stride + j];
    }
    if (returned) {
        __threadfence_block();
        __syncthreads();
    }

    // every row's place and position; the row that opens a new page enters it into the table
    uint32_t faults = 0;
    for (int i0 = tid; i0 < a.max_rows; i0 += kRowsAtOnce * T) {
        int i[kRowsAtOnce], r[kRowsAtOnce], p[kRowsAtOnce], pg[kRowsAtOnce], id[kRowsAtOnce];
        int32_t *entry[kRowsAtOnce];
        bool opens[kRowsAtOnce];
#pragma unroll
        for (int e = 0; e < kRowsAtOnce; ++e) i[e] = i0 + e * T;
        upper<kRowsAtOnce>(s_row, n, i, r);
#pragma unroll
        for (int e = 0; e < kRowsAtOnce; ++e) {
            opens[e] = false;
            id[e] = -1;
            if (i[e] >= rows) continue;
            const int l = s_len[r[e]], held = (l + ps - 1) / ps;
            p[e] = l + i[e] - (r[e] ? s_row[r[e] - 1] : 0);
            pg[e] = page_of(a.map, p[e]);
            entry[e] = a.table + (size_t)r[e] * a.table_stride + pg[e];
            opens[e] = pg[e] >= held && p[e] == pg[e] * ps;
            id[e] = pg[e] < held ? *entry[e] : a.free_pages[F1 - 1 - (s_new0[r[e]] + pg[e] - held)];
        }
#pragma unroll
        for (int e = 0; e < kRowsAtOnce; ++e) {
            if (i[e] >= a.max_rows) continue;
            int slot = -1, pos = 0;
            if (i[e] < rows) {
                if (opens[e]) *entry[e] = id[e];
                slot = place_of(a.map, p[e], pg[e], id[e]);
                pos = a.pos0 + p[e];
                faults += slot < 0;
            }
            a.slots[i[e]] = slot;
            a.pos[i[e]] = pos;
        }
    }
    if (faults) page_fault(a.faults);
}

// RoPE of the q and k heads of each row of stacked q | k | v at the row's
// position, q to rows of its own, k and v to the row's slot, f16 values
// rounded to nearest even (rope_kv_f16_kernel's arithmetic).  A thread takes
// four rotation pairs (values d and d + head_dim/2) of a q or k head, or
// eight values of a v head, with 16-byte loads; heads of quantised caches are
// left to the block part of the grid.  Rows without a place (slot < 0) are
// left out whole.  Bound by its bytes: 1717 rows of 8 + 2 * 4 heads of 256 dims (47 MB) take 10.1 us,
// 4.7 TB/s; few rows by the launch (24 rows 2.6 us).  Without an angle table by the angles (a pow in 64 bits, a
// sine and a cosine a pair and row: 63 us for 1710 rows).
//
// The block part: one wave a pair of 32-value blocks (each half wave one), the
// value rotated by its own lane, then the reference's block quantisers
// (kv_append_any_kernel's rule).  Bound by issue: both quantisers for each value and stores of single bytes; 1710 rows
// into Q8_0 take 27 us, 1.8 TB/s, into Q4_0 26.
template <int KF, int VF>
__global__ __launch_bounds__(256) void append_paged_kernel(const float *__restrict__ qkv, float *__restrict__ q_out,
                                                           uint8_t *__restrict__ k_pages, uint8_t *__restrict__ v_pages,
                                                           const int32_t *__restrict__ slots,
                                                           const int32_t *__restrict__ positions, int n_slots,
                                                           int n_heads, int n_kv_heads, int head_dim, int item_wgs,
                                                           RopeArgs rope, uint32_t *faults)
{
    const int row = blockIdx.y, slot = slots[row], pos = positions[row];
    if (slot < 0) return;
    if (slot >= n_slots) {
        if (threadIdx.x == 0 && blockIdx.x == 0) page_fault(faults);
        return;
    }
    const int half = head_dim >> 1, width = (n_heads + 2 * n_kv_heads) * head_dim;
    const float *src = qkv + (size_t)row * width;
    const size_t k_row = (size_t)slot * n_kv_heads * kv_row_bytes(KF, head_dim);
    const size_t v_row = (size_t)slot * n_kv_heads * kv_row_bytes(VF, head_dim);
    if ((int)blockIdx.x < item_wgs) {
        const int per = head_dim >> 3;  // items a head
        const int item = blockIdx.x * 256 + threadIdx.x;
        const int head = item / per, j = item - head * per;
        if (head >= n_heads + 2 * n_kv_heads) return;
        if (head < n_heads + n_kv_heads) {
            if (KF != 0 && head >= n_heads) return;
            const float *x = src + (size_t)head * head_dim + j * 4;
            const float4 lo = *reinterpret_cast<const float4 *>(x), hi = *reinterpret_cast<const float4 *>(x + half);
            float c[4], s[4], r0[4], r1[4];
            if (rope.table && pos >= 0 && pos < rope.n_table) {
                const float2 *t = reinterpret_cast<const float2 *>(rope.table) + (size_t)pos * half + j * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 cs = t[e];
                    c[e] = cs.x;
                    s[e] = cs.y;
                }
            } else {
#pragma unroll 1
                for (int e = 0; e < 4; ++e) rope_cs(rope, pos, j * 4 + e, head_dim, c[e], s[e]);
            }
            const float v0[4] = {lo.x, lo.y, lo.z, lo.w}, v1[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r0[e] = v0[e] * c[e] - v1[e] * s[e];
                r1[e] = v0[e] * s[e] + v1[e] * c[e];
            }
            if (head < n_heads) {
                float *dst = q_out + ((size_t)row * n_heads + head) * head_dim + j * 4;
                *reinterpret_cast<float4 *>(dst) = make_float4(r0[0], r0[1], r0[2], r0[3]);
                *reinterpret_cast<float4 *>(dst + half) = make_float4(r1[0], r1[1], r1[2], r1[3]);
            } else {
                uint16_t *dst = reinterpret_cast<uint16_t *>(k_pages + k_row) + (size_t)(head - n_heads) * head_dim + j * 4;
                *reinterpret_cast<ushort4 *>(dst) = make_ushort4(f32_to_f16_rne(r0[0]), f32_to_f16_rne(r0[1]),
                                                                 f32_to_f16_rne(r0[2]), f32_to_f16_rne(r0[3]));
                *reinterpret_cast<ushort4 *>(dst + half) = make_ushort4(f32_to_f16_rne(r1[0]), f32_to_f16_rne(r1[1]),
                                                                        f32_to_f16_rne(r1[2]), f32_to_f16_rne(r1[3]));
            }
        } else if (VF == 0) {
            const float *x = src + (size_t)head * head_dim + j * 8;
            const float4 lo = *reinterpret_cast<const float4 *>(x), hi = *reinterpret_cast<const float4 *>(x + 4);
            uint16_t *dst = reinterpret_cast<uint16_t *>(v_pages + v_row) +
                            (size_t)(head - n_heads - n_kv_heads) * head_dim + j * 8;
            const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = (uint32_t)f32_to_f16_rne(v[2 * e]) | ((uint32_t)f32_to_f16_rne(v[2 * e + 1]) << 16);
            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
    if constexpr (KF != 0 || VF != 0) {
        const int nb = head_dim / 32, k_blocks = KF ? n_kv_heads * nb : 0, v_blocks = VF ? n_kv_heads * nb : 0;
        const int lane = threadIdx.x & 63, l = lane & 31;
        const int b0 = (((int)blockIdx.x - item_wgs) * 4 + (threadIdx.x >> 6)) * 2;  // the wave's two blocks
        if (b0 >= k_blocks + v_blocks) return;
        const int b = b0 + (lane >> 5);
        const bool live = b < k_blocks + v_blocks, is_k = b < k_blocks;
        const int kb = live ? (is_k ? b : b - k_blocks) : 0, head = kb / nb, d = (kb - head * nb) * 32 + l;
        float v = 0.0f;
        if (live && is_k) {
            const float *x = src + (size_t)(n_heads + head) * head_dim;
            const int i = d < half ? d : d - half;
            float c, s;
            rope_cs(rope, pos, i, head_dim, c, s);
            const float v0 = x[i], v1 = x[i + half];
            v = d < half ? v0 * c - v1 * s : v0 * s + v1 * c;
        } else if (live) {
            v = src[(size_t)(n_heads + n_kv_heads + head) * head_dim + d];
        }
        uint32_t d8, d4;
        int qsum;
        const int q8 = q8_0_block32(v, d8, qsum);
        const int q4 = q4_0_block32(v, d4);
        const int q4_hi = __shfl_down(q4, 16, 64);  // value l + 16 of the block, for l < 16
        if (!live) return;
        const int fmt = is_k ? KF : VF;
        uint8_t *blk = (is_k ? k_pages + k_row : v_pages + v_row) + (size_t)kb * (fmt == 1 ? 34 : 18);
        if (l == 0) *reinterpret_cast<uint16_t *>(blk) = (uint16_t)(fmt == 1 ? d8 : d4);
        if (fmt == 1)
            blk[2 + l] = (uint8_t)(int8_t)q8;
        else if (l < 16)
            blk[2 + l] = (uint8_t)(q4 | (q4_hi << 4));
    }
}

int launch_append_paged(mrml_hip_ctx *ctx, const float *qkv, float *q, void *k, void *v, const int32_t *slots,
                        const int32_t *pos, int n_rows, int n_slots, int n_heads, int n_kv_heads, int head_dim,
                        int k_fmt, int v_fmt, const RopeArgs &rope)
{
    const int items = (n_heads + 2 * n_kv_heads) * (head_dim / 8), item_wgs = (items + 255) / 256;
    const int blocks = ((k_fmt != 0) + (v_fmt != 0)) * n_kv_heads * (head_dim / 32);
    uint8_t *kp = reinterpret_cast<uint8_t *>(k), *vp = reinterpret_cast<uint8_t *>(v);
    for (int first = 0; first < n_rows; first += 65535) {  // grid y
        const dim3 grid(item_wgs + (blocks + 7) / 8, std::min(65535, n_rows - first));
        const float *src = qkv + (size_t)first * (n_heads + 2 * n_kv_heads) * head_dim;
        float *dst = q + (size_t)first * n_heads * head_dim;
#define APPEND(KF, VF)                                                                                            \
    hipLaunchKernelGGL((append_paged_kernel<KF, VF>), grid, dim3(256), 0, ctx->stream, src, dst, kp, vp,          \
                       slots + first, pos + first, n_slots, n_heads, n_kv_heads, head_dim, item_wgs, rope,        \
                       ctx->d_page_faults)
        switch (k_fmt * 3 + v_fmt) {
        case 0: APPEND(0, 0); break;
        case 1: APPEND(0, 1); break;
        case 2: APPEND(0, 2); break;
        case 3: APPEND(1, 0); break;
        case 4: APPEND(1, 1); break;
        case 5: APPEND(1, 2); break;
        case 6: APPEND(2, 0); break;
        case 7: APPEND(2, 1); break;
        default: APPEND(2, 2); break;
        }
#undef APPEND
        if (int rc = check_launch(ctx, "append_paged_kernel")) return rc;
    }
    return MRML_HIP_OK;
}

// What the three entry points ask of a paged cache's sizes.
int pages_ok(mrml_hip_ctx *ctx, const char *name, int32_t n_pages, int32_t page_size)
{
    REQUIRE(ctx, page_size >= 1 && page_size <= kMaxPageSize, "%s: page_size=%d (1..%d)", name, page_size, kMaxPageSize);
    REQUIRE(ctx, n_pages >= 1 && (int64_t)n_pages * page_size <= INT32_MAX, "%s: n_pages=%d of %d rows (at least one, "
            "below 2^31 rows in all)", name, n_pages, page_size);
    return MRML_HIP_OK;
}

int table_ok(mrml_hip_ctx *ctx, const char *name, int32_t n_seqs, int32_t table_stride, int32_t page_size,
             int32_t max_rows)
{
    REQUIRE(ctx, n_seqs >= 1 && n_seqs <= kMaxSeqs, "%s: n_seqs=%d (1..%d)", name, n_seqs, kMaxSeqs);
    REQUIRE(ctx, table_stride >= 1 && (int64_t)table_stride * page_size <= kMaxTablePositions,
            "%s: table_stride=%d pages of %d rows (at least one, at most %d rows)", name, table_stride, page_size,
            kMaxTablePositions);
    REQUIRE(ctx, max_rows >= 1 && max_rows <= (1 << 20), "%s: max_rows=%d (1..2^20)", name, max_rows);
    return MRML_HIP_OK;
}

int formats_ok(mrml_hip_ctx *ctx, const char *name, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
               int32_t k_format, int32_t v_format)
{
    if (k_format < 0 || k_format > 2 || v_format < 0 || v_format > 2)
        return fail(ctx, MRML_HIP_E_UNSUPPORTED, "%s: k_format=%d v_format=%d (0 f16, 1 Q8_0, 2 Q4_0)", name,
                    k_format, v_format);
    REQUIRE(ctx, n_heads > 0 && n_heads <= 4096 && n_kv_heads > 0 && n_heads % n_kv_heads == 0,
            "%s: n_heads=%d n_kv_heads=%d", name, n_heads, n_kv_heads);
    REQUIRE(ctx, attn_any_ok(n_heads, n_kv_heads, head_dim),
            "%s: head_dim=%d (a multiple of 32 up to 512), group %d (at most 16)", name, head_dim,
            n_heads / n_kv_heads);
    return MRML_HIP_OK;
}

// Whether n floats at x and m floats at y share memory.
bool overlap(const float *x, size_t n, const float *y, size_t m)
{
    return (uintptr_t)x < (uintptr_t)(y + m) && (uintptr_t)y < (uintptr_t)(x + n);
}

}  // namespace

}  // namespace mrml

using namespace mrml;

extern "C" {

int mrml_hip_block_tables(mrml_hip_ctx *ctx, const int32_t *lens, const int32_t *want, int32_t n_seqs, int32_t *table,
                          int32_t table_stride, int32_t page_size, int32_t *free_pages, const int32_t *n_free,
                          int32_t n_pages, int32_t *lens_out, int32_t *n_free_out, int32_t *row_start, int32_t *slots,
                          int32_t *pos, int32_t max_rows, int32_t *status, int32_t pos0)
{
    CTX_GUARD(ctx);
    REQUIRE(ctx, lens && want && table && free_pages && n_free && lens_out && n_free_out && row_start && slots && pos &&
                     status, "block_tables: null pointer");
    if (int rc = pages_ok(ctx, "block_tables", n_pages, page_size)) return rc;
    if (int rc = table_ok(ctx, "block_tables", n_seqs, table_stride, page_size, max_rows)) return rc;
    REQUIRE(ctx, pos0 >= 0 && pos0 <= kMaxTablePositions, "block_tables: pos0=%d (0..%d)", pos0, kMaxTablePositions);
    const BlockTablesArgs a{lens, want, table, free_pages, n_free, lens_out, n_free_out, row_start, slots, pos, status,
                            n_seqs, table_stride, max_rows, pos0, page_map(n_pages, page_size), ctx->d_page_faults};
    // one thread a request or row, whichever are more, up to the workgroup
    const int threads = std::min(kTablesT, (std::max(n_seqs, max_rows) + 63) / 64 * 64);
    const int t = std::max(threads, (n_seqs + kTablesPer * 64 - 1) / (kTablesPer * 64) * 64);
    hipLaunchKernelGGL(block_tables_kernel, dim3(1), dim3(t), (size_t)n_seqs * 16, ctx->stream, a);
    return check_launch(ctx, "block_tables_kernel");
}

int mrml_hip_rope_kv_append_paged(mrml_hip_ctx *ctx, const float *qkv, float *q, uint16_t *k_pages, uint16_t *v_pages,
                                  const int32_t *slots, const int32_t *pos, int32_t n_rows, int32_t n_pages,
                                  int32_t page_size, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                  float freq_base, float freq_scale, int32_t k_format, int32_t v_format,
                                  const float *d_table, int32_t n_table)
{
    CTX_GUARD(ctx);
    const char *name = "rope_kv_append_paged";
    REQUIRE(ctx, qkv && q && k_pages && v_pages && slots && pos, "%s: null pointer", name);
    if (int rc = formats_ok(ctx, name, n_heads, n_kv_heads, head_dim, k_format, v_format)) return rc;
    if (int rc = pages_ok(ctx, name, n_pages, page_size)) return rc;
    REQUIRE(ctx, n_rows >= 1 && n_rows <= (1 << 20), "%s: n_rows=%d (1..2^20)", name, n_rows);
    const size_t q_dim = (size_t)n_heads * head_dim, width = (size_t)(n_heads + 2 * n_kv_heads) * head_dim;
    REQUIRE(ctx, !overlap(q, n_rows * q_dim, qkv, n_rows * width), "%s: q must not share memory with the stacked rows",
            name);
    REQUIRE(ctx, ((((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0),
            "%s: pointers must be 16-byte aligned", name);
    REQUIRE(ctx, ((uintptr_t)d_table & 7) == 0 && n_table >= 0, "%s: table", name);
    return launch_append_paged(ctx, qkv, q, k_pages, v_pages, slots, pos, n_rows, n_pages * page_size, n_heads,
                               n_kv_heads, head_dim, k_format, v_format,
                               rope_args(d_table, n_table, freq_base, freq_scale, nullptr));
}

int mrml_hip_attention_paged(mrml_hip_ctx *ctx, const float *q, int32_t q_stride, const uint16_t *k_pages,
                             const uint16_t *v_pages, float *out, int32_t n_pages, int32_t page_size,
                             const int32_t *prefix, int32_t prefix_len, const int32_t *table, int32_t table_stride,
                             const int32_t *lens, const int32_t *row_start, int32_t n_seqs, int32_t max_rows,
                             int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                             int32_t sliding_window, int32_t k_format, int32_t v_format)
{
    CTX_GUARD(ctx);
    const char *name = "attention_paged";
    REQUIRE(ctx, q && k_pages && v_pages && out && table && lens && row_start && (prefix || prefix_len == 0),
            "%s: null pointer", name);
    if (int rc = formats_ok(ctx, name, n_heads, n_kv_heads, head_dim, k_format, v_format)) return rc;
    if (int rc = pages_ok(ctx, name, n_pages, page_size)) return rc;
    if (int rc = table_ok(ctx, name, n_seqs, table_stride, page_size, max_rows)) return rc;
    REQUIRE(ctx, prefix_len >= 0 && prefix_len <= kMaxTablePositions, "%s: prefix_len=%d (0..%d)", name, prefix_len,
            kMaxTablePositions);
    REQUIRE(ctx, q_stride >= n_heads * head_dim && q_stride % 4 == 0,
            "%s: q_stride=%d (a multiple of 4, at least n_heads * head_dim = %d)", name, q_stride, n_heads * head_dim);
    REQUIRE(ctx, ((((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) == 0),
            "%s: pointers must be 16-byte aligned", name);
    REQUIRE(ctx, std::isfinite(scale), "%s: scale=%g", name, (double)scale);
    PagedAttn a{};
    a.q = q;
    a.k = reinterpret_cast<const uint8_t *>(k_pages);
    a.v = reinterpret_cast<const uint8_t *>(v_pages);
    a.out = out;
    a.prefix = prefix;
    a.table = table;
    a.lens = lens;
    a.row_start = row_start;
    a.faults = ctx->d_page_faults;
    a.map = page_map(n_pages, page_size);
    a.q_stride = q_stride;
    a.prefix_len = prefix_len;
    a.table_stride = table_stride;
    a.n_seqs = n_seqs;
    a.max_rows = max_rows;
    a.n_heads = n_heads;
    a.n_kv_heads = n_kv_heads;
    a.head_dim = head_dim;
    a.group = n_heads / n_kv_heads;
    a.group_magic = a.group > 1 ? (uint32_t)((1ull << 32) / a.group) + 1u : 0u;
    a.longest = table_stride * page_size;
    a.window = sliding_window > 0 ? std::min(sliding_window, 2 * kMaxTablePositions) : 0;  // no row sees more
    a.k_fmt = k_format;
    a.v_fmt = v_format;
    a.scale = scale;
    REQUIRE(ctx, paged_attn_countable(a),
            "%s: n_seqs=%d, max_rows=%d and positions (%d of a table row, prefix %d) are too many for one call", name, n_seqs,
            max_rows, a.longest, prefix_len);
    // The joining launch may read a row and head of q again before it writes the same of out, in any order of them.
    const size_t q_dim = (size_t)n_heads * head_dim, q_span = (size_t)(max_rows - 1) * q_stride + q_dim;
    REQUIRE(ctx, !overlap(out, max_rows * q_dim, q, q_span) || (out == q && (size_t)q_stride == q_dim),
            "%s: out shares memory with q (it may be q itself where the rows of q are not apart)", name);
    void *scratch = workspace(ctx, std::max<size_t>(paged_attn_scratch_bytes(a), 16));
    if (!scratch) return MRML_HIP_E_ALLOC;
    return launch_paged_attn(ctx, a, scratch);
}

}  // extern "C"
