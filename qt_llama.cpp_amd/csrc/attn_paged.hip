// attn_paged.hip -- attention of a batch of requests over a paged KV cache
// and a prefix that all of them share.
//
// Row i of request r stands at own position lens[r] - rows(r) + i, behind the
// prefix; it sees the prefix and its request's own positions up to itself,
// the last `window` of them.  out = sum_t p_t v_t with p = softmax over the
// seen t of scale * q . k_t.
//
// The softmax is taken apart over positions: any range of them gives (m, l, o)
// = (max, sum of 2^(x - m), sum of 2^(x - m) v) with x = log2(e) * scale * q.k,
// and ranges join exactly as sum 2^(m_i - M) (l_i, o_i).  So the work is a list
// of items -- (a tile of query rows that share their K and V: 16 of a stream item, 64 to
// 256 of a block item) x (a kv head) x (the positions of the prefix or of one request) -- cut
// into units of positions and dealt out evenly to 256 workgroups; paged_merge_kernel joins the
// parts.  The prefix's K and V are read once for a tile of all requests' rows, not once a request.
//
// Query rows of one kv head (every head of its group, every row of a request,
// and for the prefix every row of the batch) are the columns of the matrix
// products: S^T = K q^T and o^T = V^T p^T on 16x16x32 f16 MFMA.  K and V are f16
// exactly; q and p are f32 and enter as two f16 terms each (hi = the value
// rounded, lo = the rest rounded: 22 bits), since one f16 term would cost 2^-12
// relative and the framework's tolerance is 1e-5.  That doubles the matrix
// work; a row of q is scaled by a power of two and p by 2^14 so that no term
// falls below f16's range.  Both products leave a lane with one query row (its
// lane % 16), so row statistics need no exchange beyond the row maximum.

#include <algorithm>
#include <type_traits>

#include "any_bytes.h"
#include "paged.h"

namespace mrml {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef int int4v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kShift = 14.0f;   // p is kept as p * 2^14 (below 2^16, f16's end, with the slack below)
constexpr float kSlack = 1.5f;    // the maximum may grow by this much before o and l are rescaled
constexpr float kBroken = -1.0f;  // in place of l: the part is no good (see usable)
// Largest maximum (log2 domain, either sign) that a part may have.  p = 2^(fma(x, c, 14 - m)) is off by what the
// roundings of m and of 14 - m leave in the exponent, half a step of m each: 2^-4 in all here, so p stays below
// f16's end with the slack, and l and o share the error.  Beyond 2^24 a weight of 1 comes out as 2^6 or as nothing.
constexpr float kFarScore = 0x1p20f;
constexpr int kRowsA = 16, kUnitA = 32;  // rows and positions of a stream item's tile (one wave)
// Groups of at most so many rows are stream items (two waves' K and V come from memory or L2 twice; a block's rows
// past the group's idle).  Lines of 16 | 32 | 64: 16 requests of 24 rows behind nothing, 2000 positions of 8 heads of
// 128 dims 79 | 67 | 67 us, of 32 rows of 64 dims 60 | 46 | 46; 32 requests (64 rows) behind 4001 positions - | 34 | 42.
constexpr int kFewRows = 32;
// Costs for the split of the work.  A stream item's own cost (q, the first K and V, the part's store: a chain of
// round trips) in its units; a block unit in stream units of one wave, per 32 rows of it and wave; a block item's own
// cost is a time too (q and the first tiles in, o out: as many bytes at every head size), in units that take as long
// as they have rows.  Measured on both sides, us:
//   stream item 1 | 2 | 4: 32 requests behind 4001 positions 36.0 | 34.0 | 34.7, 20 of up to 30000 82.5 | 82.3 | 81.4
//   block unit 0.1 | 0.15 | 0.22: 256 requests behind 32768 positions 234 | 223 | 238, 32 behind 4001 33.0 | 34.0 | 35.9
//   block item of 128 rows 2 | 3 | 4 | 6: 11 chunks behind 3000 positions 183 | 172 | 160 | 166, 100 of 1..100 rows
//   behind 3000 171 | 164 | 152 | 162; of 256 rows 2 | 3 | 4 | 6: 4 chunks of 500 behind 2000 249 | 251 | 259 | 268
constexpr int kItemCost = 2;
constexpr float kBlockCost = 0.15f;
constexpr int block_item_cost(int rows) { return rows ? 512 / rows : 0; }

// Waves of a workgroup, rows of a block item and positions of its tile by padded head size: two waves a SIMD
// while a wave's q and o fit 256 registers.
constexpr int waves_of(int dp, int kf, int vf)
{
    return dp > 256 && vf && !kf ? 2 : dp > (kf || vf ? 128 : 256) ? 4 : 8;  // 2: both tiles of 4 would not fit LDS
}
constexpr int tiles_of(int dp) { return dp > 128 ? 1 : 2; }  // row tiles of 16 a wave
constexpr int rows_b(int dp) { return waves_of(dp, 0, 0) * tiles_of(dp) * 16; }
constexpr int unit_b(int dp) { return 16384 / dp; }

// Device scratch of a call (paged_attn_scratch_bytes).
struct Parts {
    float *o[2];         // first part of each row's prefix and own item: [row][head][head_dim]
    float2 *ml[2];       // (m, l) of those
    float *o_a, *o_b;    // later parts, by worker: [worker][16][head_dim], [workgroup][rows_b][head_dim]
    float2 *ml_a, *ml_b;
    int32_t *first, *last;  // workers that hold an item's first and last unit
    int4 *row_item;         // of a row: {request, its first row, its rows}
    int32_t *head;          // {the row starts are sound, first row, end of rows}
    // Items are numbered with gaps, so that nothing has to count them: a request's row tiles by its first row and
    // its place in the batch ((first row * group) / tile rows + r + tile), the prefix's behind them; times n_kv_heads.
    int pre_a, own_b, pre_b;  // the first stream item of the prefix, block item of a request, of the prefix
    int wgs, waves;
    int rows_b;               // rows of a block item (0: none)
};

// What a wave knows of the piece it works on (uniform).
struct Piece {
    const int32_t *table;
    int p0, p1;        // positions of this piece, in the source's own count
    int row0, rows;    // first query row of the tile and number of rows in the group
    int tok0;          // first token row of the group
    int at0;           // own position of the group's first token (own items)
    int kvh;
    bool pre;          // the prefix
};

// Where a piece's part goes: to its rows' own places (the item's first part), or to its worker's.
struct Dest {
    float *o;
    float2 *ml;
    bool own;
};

template <int T>
struct Scan {  // over the requests, in LDS
    int ua[T + 1], ub[T + 1];  // stream and block units before each thread's share of the requests
    int rs[T + 1], len[T];     // the share's first row, its first request's length
    int sum[8][2], low[8], flags[8];
};

__device__ __forceinline__ float as_f(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_u(float f) { return __builtin_bit_cast(uint32_t, f); }

// Lane l's value joined with those of lanes l ^ 16, l ^ 32, l ^ 48 (the lanes of one query row).
template <class F>
__device__ __forceinline__ float over_row(float v, F f)
{
    const auto a = __builtin_amdgcn_permlane16_swap(as_u(v), as_u(v), false, false);
    v = f(as_f(a[0]), as_f(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(as_u(v), as_u(v), false, false);
    return f(as_f(b[0]), as_f(b[1]));
}
__device__ __forceinline__ float row_max(float v) { return over_row(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float row_sum(float v) { return over_row(v, [](float a, float b) { return a + b; }); }

// A value that every lane of the wave holds, as a scalar.
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// No memory access is moved past this by the compiler (waits that count loads rely on their order).
__device__ __forceinline__ void pin()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// What lanes of this wave wrote to LDS before is there for its other lanes after (a wave's LDS accesses keep their
// order; the barrier alone tells the compiler nothing about memory).
__device__ __forceinline__ void wave_handover()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// v, as a value that the compiler forms anew where it is used: what follows from it is
// not kept in registers across a loop.
__device__ __forceinline__ int here(int v)
{
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float kv_value(const uint8_t *row, int fmt, int d)
{
    if (fmt == 0) return f16_bits_to_f32(reinterpret_cast<const uint16_t *>(row)[d]);
    const uint8_t *b = row + (size_t)(d >> 5) * (fmt == 1 ? 34 : 18);
    const float s = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(b));
    const int l = d & 31;
    if (fmt == 1) return s * (float)(int8_t)b[2 + l];
    const int x = b[2 + (l & 15)];
    return s * (float)((l < 16 ? x & 15 : x >> 4) - 8);
}

__device__ __forceinline__ int place_at(const PagedAttn &a, const int32_t *table, int pos)
{
    const int pg = page_of(a.map, pos);
    return place_of(a.map, pos, pg, table[pg]);
}

// The rows of one kv head in a cache: place p's at base + p * stride.
struct HeadRows {
    const uint8_t *base;
    uint32_t stride;
    __device__ __forceinline__ const uint8_t *row(int place) const
    {
        return base + (uint64_t)(uint32_t)max(place, 0) * stride;  // none: the first, which is there
    }
};

__device__ __forceinline__ HeadRows head_rows(const PagedAttn &a, const uint8_t *cache, int fmt, int kvh)
{
    const int bytes = kv_row_bytes(fmt, a.head_dim);
    return HeadRows{cache + (size_t)kvh * bytes, (uint32_t)(a.n_kv_heads * bytes)};
}

// ---- the requests' shares of the work --------------------------------------------

// All workgroups do this first, out of cold instruction caches: what counts is
// the number of instructions, so divisions are by multiplication and sums over the
// lanes by DPP.

struct Request {
    int rs, n, len;  // first row, rows, own length (within its table row)
};

__device__ __forceinline__ int div_group(const PagedAttn &a, int x)  // x * group < 2^32
{
    return a.group_magic ? (int)__umulhi((uint32_t)x, a.group_magic) : x;
}

// x / y for 0 <= x < 2^30, y > 0: the reciprocal's quotient, then its remainder's, then what a rounding left.
__device__ __forceinline__ int div_fast(int x, int y, int &rest)
{
    const float inv = __builtin_amdgcn_rcpf((float)y);
    int q = (int)((float)x * inv);
    int r = x - q * y;
    const int d = (int)((float)r * inv);
    q += d;
    r -= d * y;
    if (r < 0) --q, r += y;
    if (r >= y) ++q, r -= y;
    rest = r;
    return q;
}

template <int T>
__device__ __forceinline__ int share(const PagedAttn &a) { return (a.n_seqs + T - 1) / T; }

__device__ __forceinline__ int clamp_len(const PagedAttn &a, int len) { return min(max(len, 0), a.longest); }

template <int T>
__device__ __forceinline__ Request request_at(const PagedAttn &a, const Scan<T> &s, int r)
{
    if (share<T>(a) == 1) return Request{s.rs[r], s.rs[r + 1] - s.rs[r], s.len[r]};
    const int rs = a.row_start[r];
    return Request{rs, a.row_start[r + 1] - rs, clamp_len(a, a.lens[r])};
}

// Own positions that the rows of a request up to row i1, from row i0 on, see: [lo, hi).
__device__ __forceinline__ void own_range(const PagedAttn &a, const Request &q, int i0, int i1, int &lo, int &hi)
{
    hi = max(q.len - q.n + i1 + 1, 0);
    lo = a.window ? min(max(q.len - q.n + i0 - a.window + 1, 0), hi) : 0;
}

// The same of a row tile of a request.
template <int TILE>
__device__ __forceinline__ void tile_range(const PagedAttn &a, const Request &q, int tile, int &lo, int &hi)
{
    own_range(a, q, div_group(a, tile * TILE), div_group(a, min(q.n * a.group, (tile + 1) * TILE) - 1), lo, hi);
}

template <int UNIT>
__device__ __forceinline__ int units_of(int lo, int hi) { return max(1, (hi - lo + UNIT - 1) / UNIT); }

// The units of a request, with each item's own cost: of stream items (all its row
// tiles take the positions that any of its rows sees) or of block items.
template <int ROWS, int UNIT>
__device__ __forceinline__ void request_units(const PagedAttn &a, const Request &q, int &ua, int &ub)
{
    ua = ub = 0;
    if (q.n <= 0) return;
    const int m = q.n * a.group;
    int lo, hi;
    if (!ROWS || m <= kFewRows) {
        own_range(a, q, 0, q.n - 1, lo, hi);
        ua = (m + kRowsA - 1) / kRowsA * a.n_kv_heads * (units_of<kUnitA>(lo, hi) + kItemCost);
    } else if constexpr (ROWS != 0) {
        for (int b = 0; b * ROWS < m; ++b) {
            tile_range<ROWS>(a, q, b, lo, hi);
            ub += units_of<UNIT>(lo, hi) + block_item_cost(ROWS);
        }
        ub *= a.n_kv_heads;
    }
}

// Inclusive sum over a wave's lanes.
__device__ __forceinline__ int wave_scan(int x)
{
#define SCAN_STEP(CTRL, ROWS) x += __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false)
    SCAN_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
    SCAN_STEP(0x112, 0xf);
    SCAN_STEP(0x114, 0xf);
    SCAN_STEP(0x118, 0xf);
    SCAN_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    SCAN_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef SCAN_STEP
    return x;
}

struct Totals {
    bool ok, need_at;  // the row starts ascend within the rows; some row stands before its request's first position
    int low;           // with a window: the first own position that a row has
};

template <int T, int ROWS, int UNIT>
__device__ __forceinline__ Totals scan_requests(const PagedAttn &a, Scan<T> &s)
{
    const int tid = threadIdx.x, wave = tid >> 6;
    const int per = share<T>(a), r0 = min(tid * per, a.n_seqs), r1 = min(r0 + per, a.n_seqs);
    int w[2] = {0, 0}, low = INT32_MAX;
    bool bad = false, neg = false;
    int rs = a.row_start[r0];
    s.rs[tid] = rs;
    if (tid == T - 1) s.rs[T] = a.row_start[a.n_seqs];
    for (int r = r0; r < r1; ++r) {
        const int re = a.row_start[r + 1], len = a.lens[r];
        if (rs < 0 || re < rs || re > a.max_rows) {
            bad = true;
        } else {
            const Request q{rs, re - rs, clamp_len(a, len)};
            if (q.len != len && blockIdx.x == 0) page_fault(a.faults);
            if (r == r0) s.len[tid] = q.len;
            int ua, ub;
            request_units<ROWS, UNIT>(a, q, ua, ub);
            w[0] += ua;
            w[1] += ub;
            if (q.n > 0) {
                low = min(low, q.len - q.n);
                neg |= q.len < q.n;
            }
        }
        rs = re;
    }
    const int inc[2] = {wave_scan(w[0]), ROWS ? wave_scan(w[1]) : 0};
    const int flags = (__any(bad) ? 1 : 0) | (__any(neg) ? 2 : 0);
    if (a.window)
        for (int d = 32; d; d >>= 1) low = min(low, __shfl_xor(low, d, 64));
    if ((tid & 63) == 63) {
        s.sum[wave][0] = inc[0];
        s.sum[wave][1] = inc[1];
        s.low[wave] = low;
        s.flags[wave] = flags;
    }
    __syncthreads();
    int before[2] = {0, 0}, all = 0;
    low = INT32_MAX;
#pragma unroll 1
    for (int v = 0; v < T / 64; ++v) {
        if (v < wave) before[0] += s.sum[v][0], before[1] += s.sum[v][1];
        low = min(low, s.low[v]);
        all |= s.flags[v];
    }
    s.ua[tid] = before[0] + inc[0] - w[0];
    s.ub[tid] = before[1] + inc[1] - w[1];
    if (tid == T - 1) {
        s.ua[T] = before[0] + inc[0];
        s.ub[T] = before[1] + inc[1];
    }
    __syncthreads();
    all = uni(all);
    return Totals{(all & 1) == 0, (all & 2) != 0, uni(low)};
}

// The thread whose share [from[t], from[t + 1]) holds x (from ascending, from[0] <= x < from[T]).
template <int T>
__device__ __forceinline__ int share_of(const int *from, int x)
{
    int lo = 0;
#pragma unroll 1
    for (int step = T / 2; step; step >>= 1)
        if (from[lo + step] <= x) lo += step;
    return lo;
}

// The request of a row (the last one that starts at or before it and has rows).
template <int T>
__device__ __forceinline__ int request_of(const PagedAttn &a, const Scan<T> &s, int row)
{
    const int per = share<T>(a);
    int r = share_of<T>(s.rs, row) * per;
    if (per > 1)
        while (r + 1 < a.n_seqs && a.row_start[r + 1] <= row) ++r;
    return r;
}

// ---- query rows ------------------------------------------------------------------

__device__ __forceinline__ size_t part_row(const PagedAttn &a, const Piece &pc, const Dest &d, int mi)
{
    if (!d.own) return (size_t)(mi - pc.row0);
    const int i = div_group(a, mi);
    return (size_t)(pc.tok0 + i) * a.n_heads + pc.kvh * a.group + (mi - i * a.group);
}

// What row mi of a piece's group sees, in the source's positions: [vlo, vhi).
template <int T>
__device__ __forceinline__ void row_sees(const PagedAttn &a, const Scan<T> &s, bool need_at, const Piece &pc, int mi, int &vlo, int &vhi)
{
    vlo = 0;
    vhi = INT32_MAX;
    if (mi >= pc.rows) return;
    const int row = div_group(a, mi), tok = pc.tok0 + row;
    if (!pc.pre) {
        const int at = pc.at0 + row;
        vhi = at + 1;
        vlo = a.window ? at - a.window + 1 : 0;
    } else if (need_at || a.window) {
        const Request q = request_at(a, s, request_of(a, s, tok));
        const int at = a.prefix_len + q.len - (q.rs + q.n - tok);
        vhi = min(a.prefix_len, at + 1);
        vlo = a.window ? at - a.window + 1 : 0;
    }
}

__device__ __forceinline__ int wave_max(int v)
{
    for (int x = 32; x; x >>= 1) v = max(v, __shfl_xor(v, x, 64));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_min(int v) { return -wave_max(-v); }

// The factor from products to scores in the log2 domain, positive (a negative scale turns q's sign).
__device__ __forceinline__ float score_factor(const PagedAttn &a) { return fmaxf(fabsf(a.scale) * kLog2e, 0x1p-126f); }

// q of one row (or -q) as two f16 terms of q * 2^k, lane group g holding dims 32 s + 8 g ..:
// returns 2^-k.
template <int KS>
__device__ __forceinline__ float load_q(const PagedAttn &a, const float *row, bool live, int g, half8 *hi, half8 *lo)
{
    float top = 0.0f;
    float v[KS][8];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const bool in = live && s * 32 < a.head_dim;
        const float4 x = in ? *reinterpret_cast<const float4 *>(row + s * 32 + g * 8) : make_float4(0, 0, 0, 0);
        const float4 y = in ? *reinterpret_cast<const float4 *>(row + s * 32 + g * 8 + 4) : make_float4(0, 0, 0, 0);
        v[s][0] = x.x, v[s][1] = x.y, v[s][2] = x.z, v[s][3] = x.w;
        v[s][4] = y.x, v[s][5] = y.y, v[s][6] = y.z, v[s][7] = y.w;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[s][e]));
    }
    top = row_max(top);
    // the largest value into [2^13, 2^14)
    const int ex = min(max((int)(as_u(top) >> 23), 14), 254);
    const float up = as_f((uint32_t)(267 - ex) << 23) * (a.scale < 0.0f ? -1.0f : 1.0f);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = v[s][e] * up;
            const _Float16 h = (_Float16)x;
            hi[s][e] = h;
            lo[s][e] = (_Float16)(x - (float)h);
        }
    return as_f((uint32_t)(ex - 13) << 23);
}

// p (f32, at most 2^15.5) as two f16 terms, both rounded towards zero: a pair in one instruction,
// and p - hi is never negative.
__device__ __forceinline__ void split_p(float x, float y, uint32_t &hi, uint32_t &lo)
{
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    const float rx = fmaf((float)h[0], -1.0f, x), ry = fmaf((float)h[1], -1.0f, y);
    const auto l = __builtin_amdgcn_cvt_pkrtz(rx, ry);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ half8 as_half8(uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    return __builtin_bit_cast(half8, make_uint4(x, y, z, w));
}

__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Running softmax of one row: x holds N products of this lane (-inf where masked;
// a score in the log2 domain is x * c, c > 0), which become p * 2^14; m (the largest
// score) and l are brought up to date, true if o has to be multiplied by f.
template <int N>
__device__ __forceinline__ bool softmax_step(float *x, float c, float &m, float &l, float &f)
{
    float top = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
    top = row_max(top) * c;
    const bool grow = top > m + kSlack;
    f = 1.0f;
    const bool any = __any(grow);
    if (any) {
        const float m2 = grow ? top : m;
        f = grow ? exp2_hw(m - m2) : 1.0f;  // 0 from -inf
        l *= f;
        m = m2;
    }
    const float base = m == -INFINITY ? 0.0f : kShift - m;
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        x[e] = exp2_hw(fmaf(x[e], c, base));
        sum += x[e];
    }
    l += sum;
    return any;
}

// Whether a part's sums can be joined with others: they are finite (check: their sum) and its scores were near
// enough to 0 for the weights to be right.
__device__ __forceinline__ bool usable(float check, float m)
{
    return check - check == 0.0f && (m == -INFINITY || fabsf(m) < kFarScore);
}

// ---- stream items: a wave, 16 query rows, K and V straight from memory ------------
//
// Per tile of 32 positions a lane takes K of position lane % 16 (+ 16) in 16-byte
// pieces, which are the product's operand as they are, and V of 8 positions in
// 16-byte pieces of 8 dims.  V's operand wants 8 positions of one dim: an 8 x 8
// transpose inside the lane's registers, one v_perm a pair; the dims then lie
// 8 apart over the operand's rows, which only the store of o has to know.  K of
// an f16 cache goes through a tile of LDS of the wave's own (global_load_lds), so
// that the next tile's K is on its way without registers; the next V is loaded as
// soon as this one is used up.  A wave keeps a tile of K and of V on its way, eight waves of 256
// dims 256 KB a CU.  f16 caches are bound by their bytes: 256 requests of 1000 positions of 4 heads of 256 dims
// (1.05 GB) take 212 us, 4.95 TB/s of the 5.14 that a copy reaches; 4 of 32000 of 8 heads of 128 106 us.
// Quantised ones are bound by the instructions that take them apart and by the wait for LDS between
// them (VALU busy 46% of the time, LDS 40%): the latter as Q8_0 98 us (2.85 TB/s), as Q4_0 77.
//
// Quantised K is multiplied as the ring attention does it: q as Q8_0 blocks,
// each block's integer sum on the int8 MFMA (16x16x32: one block a
// step), times both scales in f32.  There q is the left operand, so that a
// lane's position, and K's scale with it, is fixed; the tile of scores changes
// sides through LDS once.  Quantised V enters as f16 terms too: d * q has at most
// 19 bits, hi = its rounding, lo = fma(d, q, -hi), both exact.

// Tiles in LDS are made of 1 KB chunks, each the left operand of one product: 16 rows
// (positions of K, dims of V) of four 16-byte pieces (8 dims, 8 positions), lane
// i + 16 g taking piece g of row i.  Row i lies at 64 * (i / 4 + 4 (i % 4)) with its
// pieces exchanged by i % 4: the 16 lanes that a wave's 16-byte reads serve together
// (0-3, 12-15, 20-23, 24-27 and so on) then meet 16 different places of the
// 64 banks, as do the eight of any eight neighbours, and 16 lanes that write one
// run of 4 x 4 dims.  Padded rows (16 bytes a row) had 4 conflict cycles a read.  A
// lane's address is one base plus a constant for every chunk.
constexpr int kChunk = 1024;

__device__ __forceinline__ int chunk_offset(int i, int g) { return ((i >> 2) + 4 * (i & 3)) * 64 + (g ^ (i & 3)) * 16; }
// what a lane of a wave's global_load_lds (which writes 16 bytes a lane, in lane order) loads
__device__ __forceinline__ int chunk_row(int lane) { return 4 * ((lane >> 2) & 3) + (lane >> 4); }
__device__ __forceinline__ int chunk_piece(int lane) { return (lane & 3) ^ (lane >> 4); }

__device__ __forceinline__ half8 read16(const uint8_t *p) { return __builtin_bit_cast(half8, *reinterpret_cast<const uint4 *>(p)); }

// ONCE: with the non-temporal hint.
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(const uint8_t *src, uint8_t *dst)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)src,
                                     (__attribute__((address_space(3))) uint32_t *)dst, 16, 0, ONCE ? 2 : 0);
}

struct __attribute__((packed, aligned(2))) Bytes8 {
    uint32_t a, b;
};

constexpr int kTrRow = 36;  // floats a query row of the score tile in LDS

constexpr int block_bytes(int fmt) { return fmt == 1 ? 34 : 18; }

// A tile of a quantised cache: 32 rows as they lie in memory.  A wave fetches them in
// 16-byte pieces, neighbouring lanes neighbouring pieces, and picks the blocks out of LDS: lanes that
// fetch their 8 bytes of a block each make an access to the cache each (1578 a tile of 32
// positions of 128 dims, 94% of the time the caches could take them in).  A row's last piece
// ends with the row.  Rows are an odd number of 32 bytes apart: 8 of them fill the 64 banks.
template <int DP, int FMT, int ALIGN>
struct QuantTile {
    static constexpr int kRow = ((DP / 32 * block_bytes(FMT) + ALIGN - 1) / ALIGN | 1) * ALIGN;
    static constexpr int kPieces = (DP / 32 * block_bytes(FMT) + 15) / 16;  // of a row, at most
    static constexpr int kLoads = (32 * kPieces + 63) / 64;
    alignas(16) uint8_t b[32 * kRow + 16];  // words around a block's quants may end behind the last row
};

struct __attribute__((packed, aligned(2))) Bytes16 {
    uint32_t x, y, z, w;
};

// A wave's pieces of such a tile: where they lie and, on their way, what they hold.
template <class TILE>
struct QuantPieces {
    using Tile = TILE;
    uint32_t at[Tile::kLoads];  // row << 16 | byte in it
    uint4 x[Tile::kLoads];
    __device__ __forceinline__ void start(int row_bytes, int lane)
    {
        const int pieces = (row_bytes + 15) / 16;
        int rest;
        const int step_row = 64 / pieces, step = 64 - step_row * pieces;
        int row = div_fast(lane, pieces, rest);
#pragma unroll
        for (int e = 0; e < Tile::kLoads; ++e) {  // past the tile: its last piece once more
            at[e] = row < 32 ? (uint32_t)row << 16 | (uint32_t)min(rest * 16, row_bytes - 16) : 31u << 16 | (uint32_t)(row_bytes - 16);
            row += step_row;
            rest += step;
            if (rest >= pieces) rest -= pieces, ++row;
        }
    }
    __device__ __forceinline__ void load(const HeadRows &rows, int place)
    {
#pragma unroll
        for (int e = 0; e < Tile::kLoads; ++e) {
            const Bytes16 y = *reinterpret_cast<const Bytes16 *>(rows.row(__shfl(place, at[e] >> 16, 64)) + (at[e] & 0xffff));
            x[e] = make_uint4(y.x, y.y, y.z, y.w);
        }
    }
    // LDS takes an access apart whose address is no multiple of its size (28 cycles each): a last piece that ends
    // with its row is written in what both share.
    __device__ __forceinline__ void store(Tile &tile, int row_bytes) const
    {
        typedef volatile __attribute__((address_space(3))) Any32 *Words;
        typedef volatile __attribute__((address_space(3))) Any16 *Halves;
        if ((row_bytes & 15) == 0) {
#pragma unroll
            for (int e = 0; e < Tile::kLoads; ++e) *reinterpret_cast<Any128 *>(tile.b + place(e)) = Any128{x[e].x, x[e].y, x[e].z, x[e].w};
        } else if ((row_bytes & 3) == 0) {
#pragma unroll
            for (int e = 0; e < Tile::kLoads; ++e) {
                const uint32_t w[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) ((Words)(tile.b + place(e)))[j] = w[j];
            }
        } else {
#pragma unroll
            for (int e = 0; e < Tile::kLoads; ++e) {
                const uint32_t w[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) ((Halves)(tile.b + place(e)))[j] = (uint16_t)(w[j / 2] >> 16 * (j & 1));
            }
        }
    }
    __device__ __forceinline__ int place(int e) const { return (at[e] >> 16) * Tile::kRow + (at[e] & 0xffff); }
};
// 8 bytes at p + at, at even: of the words around them.
__device__ __forceinline__ Bytes8 pick8(const uint8_t *p, int at)
{
    const uint8_t *w = p + (at & ~2);
    const uint32_t w0 = get32(w), w1 = get32(w + 4), w2 = get32(w + 8);
    return Bytes8{__builtin_amdgcn_alignbyte(w1, w0, at & 2), __builtin_amdgcn_alignbyte(w2, w1, at & 2)};
}

struct None {};

// Scales and sums of q's blocks: in registers, but for heads of more than 256 dims in LDS, where with them a wave's
// registers spill more (30 requests behind 4000 positions of 2 heads of 512 dims, Q4_0: 108 us so and 70 from LDS; 64
// of 2000 positions, Q8_0: 394 and 364).
constexpr bool q_scales_in_lds(int dp) { return dp > 256; }

template <int DP, int KF, int VF>
struct WaveLds {
    int place[VF ? 1 : 32];
    alignas(16) uint8_t k[KF ? 16 : DP / 16 * kChunk];  // 32 positions: chunks of 32 dims, of 16 positions
    float scores[KF ? 16 * kTrRow : 1];
    alignas(16) float q_d[KF && q_scales_in_lds(DP) ? DP / 2 : 4];  // [block][row]
    alignas(16) int q_sum8[KF == 2 && q_scales_in_lds(DP) ? DP / 2 : 4];
    std::conditional_t<KF != 0, QuantTile<DP, KF ? KF : 1, 16>, None> kq;
    std::conditional_t<VF != 0, QuantTile<DP, VF ? VF : 1, 32>, None> vq;
};

// Query rows for a quantised K: operand bytes, and scale and sum of each block
// for the four rows that this lane's results belong to.
template <int KS, bool IN_LDS>
struct QuantQ {
    long q[KS];
    float4v d[IN_LDS ? 1 : KS];
    int4v sum8[IN_LDS ? 1 : KS];  // -8 * sum of the block's quants: what Q4_0's offset takes away
};

template <int KS, int KF, bool IN_LDS>
__device__ __forceinline__ void load_quant_q(const PagedAttn &a, const float *row, bool live, int g, QuantQ<KS, IN_LDS> &out,
                                             float *q_d, int *q_sum8)
{
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const bool in = live && s * 32 < a.head_dim;
        const float4 x = in ? *reinterpret_cast<const float4 *>(row + s * 32 + g * 8) : make_float4(0, 0, 0, 0);
        const float4 y = in ? *reinterpret_cast<const float4 *>(row + s * 32 + g * 8 + 4) : make_float4(0, 0, 0, 0);
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));  // NaN never wins
        top = row_max(top);
        const float scale = top / 127.0f;
        const float d = f16_bits_to_f32(f32_to_f16_trunc(scale)), id = scale != 0.0f ? 1.0f / scale : 0.0f;
        uint32_t w[2] = {0, 0};
        int sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int q = q8_0_value(v[e], id);
            sum += q;
            w[e >> 2] |= (uint32_t)(q & 0xff) << (8 * (e & 3));
        }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        out.q[s] = (long)((uint64_t)w[0] | ((uint64_t)w[1] << 32));
        const float sd = a.scale < 0.0f ? -d : d;
        if constexpr (IN_LDS) {
            const int i = threadIdx.x & 15;
            if (g == 0) {
                q_d[16 * s + i] = sd;
                if (KF == 2) q_sum8[16 * s + i] = -8 * sum;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                out.d[s][r] = __shfl(sd, 4 * g + r, 64);
                out.sum8[s][r] = KF == 2 ? -8 * __shfl(sum, 4 * g + r, 64) : 0;
            }
        }
    }
    wave_handover();
}

template <int DP, int KF, int VF, bool ONCE>
__device__ __forceinline__ void stream_item(const PagedAttn &a, const Scan<64 * waves_of(DP, KF, VF)> &sc, bool need_at, const Piece &pc,
                                            WaveLds<DP, KF, VF> &lds, const Dest &to)
{
    constexpr bool KQ = KF != 0, VQ = VF != 0;
    constexpr int KS = DP / 32, NG = DP < 128 ? 1 : DP / 128;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, hd = a.head_dim;
    const int mi = pc.row0 + i;
    const bool live = mi < pc.rows;
    const int i_row = div_group(a, mi), tok = pc.tok0 + i_row, head = pc.kvh * a.group + mi - i_row * a.group;
    const float *q_row = a.q + (size_t)tok * a.q_stride + (size_t)head * hd;
    half8 qh[KQ ? 1 : KS], ql[KQ ? 1 : KS];
    constexpr bool kFar = KQ && q_scales_in_lds(DP);
    QuantQ<KQ ? KS : 1, kFar> qq;
    float c = score_factor(a);
    if constexpr (KQ)
        load_quant_q<KS, KF, kFar>(a, q_row, live, g, qq, lds.q_d, lds.q_sum8);
    else
        c = fmaxf(c * load_q<KS>(a, q_row, live, g, qh, ql), 0x1p-126f);
    int vlo, vhi;
    row_sees(a, sc, need_at, pc, mi, vlo, vhi);
    const int full_lo = wave_max(vlo), full_hi = wave_min(vhi);
    const HeadRows k_rows = head_rows(a, a.k, a.k_fmt, pc.kvh), v_rows = head_rows(a, a.v, a.v_fmt, pc.kvh);
    constexpr int kBlkK = block_bytes(KF), kBlkV = block_bytes(VF);

    float m = -INFINITY, l = 0.0f;
    float4v o[NG][8];
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int d = 0; d < 8; ++d) o[n][d] = float4v{0, 0, 0, 0};

    // A tile's page ids are loaded two tiles ahead and looked at one tile ahead, when they are long there.
    const int base = chunk_offset(i, g);
    auto page_ids = [&](int t0) { return t0 + (lane & 31) < pc.p1 ? pc.table[page_of(a.map, t0 + (lane & 31))] : -1; };
    auto places = [&](int t0, int id) {
        const int pos = t0 + (lane & 31);
        const int place = place_of(a.map, pos, page_of(a.map, pos), id);
        if (place < 0 && pos < pc.p1 && lane < 32) page_fault(a.faults);
        return place;
    };
    std::conditional_t<KQ, QuantPieces<QuantTile<DP, KF ? KF : 1, 16>>, None> k_on_way;
    std::conditional_t<VQ, QuantPieces<QuantTile<DP, VF ? VF : 1, 32>>, None> v_on_way;
    if constexpr (KQ) {
        k_on_way.start(kv_row_bytes(KF, hd), lane);
        if (hd < DP)  // blocks past the head: scales and quants of 0
            for (int x = kv_row_bytes(KF, hd) / 2 + (lane >> 5); x < KS * kBlkK / 2; x += 2)
                put16(lds.kq.b + (lane & 31) * lds.kq.kRow + 2 * x, 0);
    }
    if constexpr (VQ) v_on_way.start(kv_row_bytes(VF, hd), lane);
    auto load_k = [&](int place) {
        if constexpr (KQ) {
            k_on_way.load(k_rows, place);
        } else {
            const int ln = here(lane), piece = chunk_piece(ln) * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint8_t *row = k_rows.row(__shfl(place, 16 * h + chunk_row(ln), 64)) + piece;
#pragma unroll
                for (int s = 0; s < KS; ++s)
                    load_to_lds<ONCE>(row + (s * 32 < hd ? s * 64 : 0), lds.k + (h * KS + s) * kChunk);
            }
        }
    };
    uint4 v[VQ ? 1 : NG][8];
    auto load_v = [&](int place) {
        if constexpr (VQ) {
            v_on_way.load(v_rows, place);
            return;
        } else {
        lds.place[lane & 31] = place;
        wave_handover();
        const int4 pa = *reinterpret_cast<const int4 *>(lds.place + 4 * g);
        const int4 pb = *reinterpret_cast<const int4 *>(lds.place + 16 + 4 * g);
        wave_handover();
        const int pl[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const int d0 = n * 128 + 8 * (here(lane) & 15), dim = d0 < hd ? d0 : 0;  // past the head: never stored
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint4 *src = reinterpret_cast<const uint4 *>(v_rows.row(pl[j]) + dim * 2);
                v[n][j] = ONCE ? load_stream16(src) : *src;
            }
        }
        }
    };
    int id_next = page_ids(pc.p0 + kUnitA);
    int place = places(pc.p0, page_ids(pc.p0));
    load_k(place);
    pin();
    load_v(place);
    for (int t0 = pc.p0; t0 < pc.p1; t0 += kUnitA) {
        const uint32_t there = (uint32_t)__ballot(place >= 0);  // bit p: position t0 + p
        const int place_next = places(t0 + kUnitA, id_next);
        id_next = page_ids(t0 + 2 * kUnitA);
        float x[8];
        if constexpr (KQ) {
            k_on_way.store(lds.kq, kv_row_bytes(KF, hd));
            wave_handover();
            if (t0 + kUnitA < pc.p1) load_k(place_next);
            float4v acc[2] = {};
            const uint8_t *rows = lds.kq.b + i * lds.kq.kRow;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                float4v qd = qq.d[kFar ? 0 : s];
                int4v sum8 = qq.sum8[kFar ? 0 : s];
                if constexpr (kFar) {
                    qd = *reinterpret_cast<const float4v *>(lds.q_d + 16 * s + 4 * g);
                    sum8 = KF == 2 ? *reinterpret_cast<const int4v *>(lds.q_sum8 + 16 * s + 4 * g) : int4v{0, 0, 0, 0};
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t *b = rows + 16 * h * lds.kq.kRow + s * kBlkK;
                    const uint8_t *quants = b + (KF == 1 ? 8 * g : 8 * (g & 1));
                    const Bytes8 w = s & 1 ? Bytes8{get32(quants + 2), get32(quants + 6)} : pick8(quants, 2);
                    uint32_t w0 = w.a, w1 = w.b;
                    if (KF == 2) {  // dims 8 g .. of the block: low nibbles, then high ones
                        w0 = (w0 >> (4 * (g >> 1))) & 0x0f0f0f0fu;
                        w1 = (w1 >> (4 * (g >> 1))) & 0x0f0f0f0fu;
                    }
                    const long kk = (long)((uint64_t)w0 | ((uint64_t)w1 << 32));
                    const int4v is = __builtin_amdgcn_mfma_i32_16x16x32_i8(qq.q[s], kk, sum8, 0, 0, 0);
                    const float dk = f16_bits_to_f32(get16(b));
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[h][r] = fmaf((float)is[r], dk * qd[r], acc[h][r]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) lds.scores[(4 * g + r) * kTrRow + 16 * h + i] = acc[h][r];
            wave_handover();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 y = *reinterpret_cast<const float4 *>(lds.scores + i * kTrRow + 16 * h + 4 * g);
                x[4 * h] = y.x, x[4 * h + 1] = y.y, x[4 * h + 2] = y.z, x[4 * h + 3] = y.w;
            }
            wave_handover();
        } else {
            // K is in LDS once no more than this tile's V (loaded after it) is on its way
            constexpr int kLeft = VQ ? 0 : NG * 8;
            __builtin_amdgcn_s_waitcnt(0x0f70 | (kLeft & 15) | (kLeft >> 4) << 14);
            pin();
            float4v acc[2][2] = {};
            half8 kk[2][2][2];  // the next two steps' pieces are on their way while two steps' products run
            auto read_k = [&](int s0) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        kk[(s0 / 2) & 1][e][h] = read16(lds.k + base + (h * KS + s0 + e) * kChunk);
            };
            read_k(0);
#pragma unroll
            for (int s = 0; s < KS; s += 2) {
                if (s + 2 < KS) read_k(s + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        acc[h][0] = mfma(kk[(s / 2) & 1][e][h], qh[s + e], acc[h][0]);
                        acc[h][1] = mfma(kk[(s / 2) & 1][e][h], ql[s + e], acc[h][1]);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[4 * h + r] = acc[h][0][r] + acc[h][1][r];
        }
        if constexpr (!KQ) {
            pin();  // K's tile has been read, and no later load passes the next one's
            if (t0 + kUnitA < pc.p1) load_k(place_next);
            pin();
        }
        uint32_t v_there = 0xff;  // bit j: this lane's position j of V
        const bool edge = t0 < full_lo || t0 + kUnitA > full_hi || there != 0xffffffffu;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int p = 16 * (e >> 2) + 4 * g + (e & 3), pos = t0 + p;
                if (pos < vlo || pos >= vhi || !((there >> p) & 1)) x[e] = -INFINITY;
            }
            // nothing is there: whatever was read must not meet a weight of 0
            v_there = (there >> (4 * g) & 15) | (there >> (16 + 4 * g) & 15) << 4;
            if constexpr (!VQ)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(v_there >> j & 1))
#pragma unroll
                        for (int n = 0; n < NG; ++n) v[n][j] = make_uint4(0, 0, 0, 0);
        }
        float f;
        if (softmax_step<8>(x, c, m, l, f)) {
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int d = 0; d < 8; ++d) o[n][d] *= f;
        }
        uint32_t ph[4], pw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split_p(x[2 * e], x[2 * e + 1], ph[e], pw[e]);
        const half8 p_hi = as_half8(ph[0], ph[1], ph[2], ph[3]), p_lo = as_half8(pw[0], pw[1], pw[2], pw[3]);
        if constexpr (VQ) {
            v_on_way.store(lds.vq, kv_row_bytes(VF, hd));
            wave_handover();
            if (t0 + kUnitA < pc.p1) load_v(place_next);
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if constexpr (VQ) {
                const int d0 = n * 128 + 8 * i, dim = d0 < hd ? d0 : 0;  // past the head: never stored
                const uint8_t *rows = lds.vq.b + 4 * g * lds.vq.kRow;
                const int scale = (dim >> 5) * kBlkV, quants = scale + 2 + (VF == 1 ? 8 * (i & 3) : 8 * (i & 1));
                Bytes8 vq[8];
                _Float16 vd[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint8_t *b = rows + (16 * (j >> 2) + (j & 3)) * lds.vq.kRow;
                    const _Float16 d = __builtin_bit_cast(_Float16, get16(b + scale));
                    vd[j] = v_there >> j & 1 ? d : (_Float16)0.0f;
                    vq[j] = pick8(b, quants);
                }
                // quants as unsigned bytes u, read as the f16 number 1024 + u, less 1024 and the bytes' offset
                constexpr bool q8 = VF == 1;
                const int sh = 4 * ((i & 3) >> 1);
                const half2v off = q8 ? half2v{(_Float16)-1152.0f, (_Float16)-1152.0f}
                                      : half2v{(_Float16)-1032.0f, (_Float16)-1032.0f};
                uint32_t w[8][2];
                half2v d2[4];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j][0] = q8 ? vq[j].a ^ 0x80808080u : (vq[j].a >> sh) & 0x0f0f0f0fu;
                    w[j][1] = q8 ? vq[j].b ^ 0x80808080u : (vq[j].b >> sh) & 0x0f0f0f0fu;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) d2[e] = half2v{vd[2 * e], vd[2 * e + 1]};
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const uint32_t sel = 0x0c040c00u + 0x00010001u * (d & 3);
                    uint32_t t[4], u[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t b = __builtin_amdgcn_perm(w[2 * e + 1][d >> 2], w[2 * e][d >> 2], sel) | 0x64006400u;
                        const half2v q2 = __builtin_bit_cast(half2v, b) + off;
                        const half2v hi = q2 * d2[e];
                        const half2v lo = __builtin_elementwise_fma(q2, d2[e], -hi);
                        t[e] = __builtin_bit_cast(uint32_t, hi);
                        u[e] = __builtin_bit_cast(uint32_t, lo);
                    }
                    const half8 v_hi = as_half8(t[0], t[1], t[2], t[3]), v_lo = as_half8(u[0], u[1], u[2], u[3]);
                    o[n][d] = mfma(v_hi, p_hi, o[n][d]);
                    o[n][d] = mfma(v_hi, p_lo, o[n][d]);
                    o[n][d] = mfma(v_lo, p_hi, o[n][d]);
                }
            } else {
                uint32_t w[8][4];  // [position][pair of dims]
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    w[j][0] = v[n][j].x, w[j][1] = v[n][j].y, w[j][2] = v[n][j].z, w[j][3] = v[n][j].w;
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
                    uint32_t t[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = __builtin_amdgcn_perm(w[2 * e + 1][d >> 1], w[2 * e][d >> 1], sel);
                    const half8 vv = as_half8(t[0], t[1], t[2], t[3]);
                    o[n][d] = mfma(vv, p_hi, o[n][d]);
                    o[n][d] = mfma(vv, p_lo, o[n][d]);
                }
            }
        }
        if constexpr (!VQ)
            if (t0 + kUnitA < pc.p1) load_v(place_next);
        wave_handover();
        place = place_next;
    }
    l = row_sum(l);
    float check = l;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int d = 0; d < 8; ++d) check += o[n][d][0] + o[n][d][1] + o[n][d][2] + o[n][d][3];
    check = row_sum(check);
    if (live) {
        const size_t at = part_row(a, pc, to, mi);
        float *dst = to.o + at * hd;
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int dim = n * 128 + 8 * (4 * g + r);  // operand row 4 g + r: dims dim + 0..7 in o[n][0..7]
                if (dim >= hd) continue;
                *reinterpret_cast<float4 *>(dst + dim) = make_float4(o[n][0][r], o[n][1][r], o[n][2][r], o[n][3][r]);
                *reinterpret_cast<float4 *>(dst + dim + 4) = make_float4(o[n][4][r], o[n][5][r], o[n][6][r], o[n][7][r]);
            }
        if (g == 0) to.ml[at] = make_float2(m - kShift, usable(check, m) ? l : kBroken);
    }
}

// ---- block items: a workgroup, many query rows, K and V through LDS -----------------
//
// Tiles of T = 16384 / DP positions, two in LDS (128 KB): while the waves work on one,
// the next is under way.  K goes to LDS directly (global_load_lds, as in a stream
// item); V is transposed on its way by the thread that has loaded 8 positions of some
// dims, and written as 16-byte runs of 8 positions.  A wave holds 16 * R rows; each
// chunk read from LDS feeds 2 * R products.
//
// Bound by issue and power: 512 rows a kv head (256 requests, groups of 2) of 4 heads of 256 dims behind 32768 positions take 186 us,
// 370 TFLOP/s of the formula and 740 with both terms of q and p, 64% of what an 8192^3 f16 matrix product of the vendor's
// library reaches here.  MFMA is busy 40% of the time, other vector instructions take 24%, a wave
// waits 34%, and the clock falls to 1.9 GHz (2.4 in stream items).  Two tiles that fill LDS (128 KB) against smaller ones: a barrier a tile, and the next tile has the whole
// tile's products to arrive in.

template <int DP>
struct BlockLds {
    static constexpr int T = unit_b(DP);
    alignas(16) uint8_t k[2][T / 16][DP / 32][kChunk];  // [16 positions][32 dims]
    alignas(16) uint8_t v[2][T / 32][DP / 16][kChunk];  // [32 positions][16 dims]
    int place[3][T];
};

template <int DP>
__device__ __forceinline__ void block_item(const PagedAttn &a, const Scan<64 * waves_of(DP, 0, 0)> &sc, bool need_at, const Piece &pc,
                                           BlockLds<DP> &lds, const Dest &to)
{
    constexpr int NW = waves_of(DP, 0, 0), R = tiles_of(DP), KS = DP / 32, NF = DP / 16, T = unit_b(DP);
    constexpr int SP = T < 64 || DP == 128 ? 32 : 64, NH = SP / 16, kAhead = 3;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4, hd = a.head_dim;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const HeadRows k_rows = head_rows(a, a.k, 0, pc.kvh), v_rows = head_rows(a, a.v, 0, pc.kvh);
    const int tiles = (pc.p1 - pc.p0 + T - 1) / T;

    // A tile's page ids are loaded two tiles ahead and put into LDS as places at the end of that tile.
    auto page_ids = [&](int tile) {
        const int pos = pc.p0 + tile * T + tid;
        return tid < T && pos < pc.p1 ? pc.table[page_of(a.map, pos)] : -1;
    };
    auto set_places = [&](int tile, int id) {
        if (tid < T) {
            const int pos = pc.p0 + tile * T + tid, place = place_of(a.map, pos, page_of(a.map, pos), id);
            if (place < 0 && pos < pc.p1) page_fault(a.faults);
            lds.place[tile % 3][tid] = place;
        }
    };
    // K: a wave's share of the chunks, whole 16-position groups or part of one's steps
    constexpr int GW = T / 16 >= NW ? T / 16 / NW : 1, SW = T / 16 >= NW ? KS : KS * (T / 16) / NW, kPartsK = GW * SW;
    auto load_k = [&](int tile, int n) {
        const int grp = T / 16 >= NW ? wave * GW + n / SW : wave * (T / 16) / NW;
        const int s = (T / 16 >= NW ? 0 : wave * SW % KS) + n % SW, ln = here(lane);
        const uint8_t *row = k_rows.row(lds.place[tile % 3][grp * 16 + chunk_row(ln)]);
        load_to_lds<false>(row + chunk_piece(ln) * 16 + (s * 32 < hd ? s * 64 : 0), lds.k[tile & 1][grp][s]);
    };
    // V: this thread's 8 dims and NV positions: a run of 8 in the products' order (run0 + 0..3, run0 + 16..19) or
    // half of one
    constexpr int NV = 32 / NW, kHalves = 8 / NV;
    const int dl = (tid / (4 * kHalves)) % (DP / 8), half = NV == 8 ? 0 : tid & 1, run = ((tid / kHalves) & 3) + tid / (DP / 2 * kHalves) * 4;
    const int run0 = (run >> 2) * 32 + (run & 3) * 4 + half * 16;
    uint32_t v[NV][4];
    auto load_v = [&](int tile, int j) {
        const uint8_t *row = v_rows.row(lds.place[tile % 3][run0 + (j >> 2) * 16 + (j & 3)]);
        const uint4 x = *reinterpret_cast<const uint4 *>(row + (dl * 8 < hd ? dl * 16 : 0));
        v[j][0] = x.x, v[j][1] = x.y, v[j][2] = x.z, v[j][3] = x.w;
    };
    auto store_v = [&](int tile) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (lds.place[tile % 3][run0 + (j >> 2) * 16 + (j & 3)] < 0)  // nothing there: no weight may meet it
#pragma unroll
                for (int w = 0; w < 4; ++w) v[j][w] = 0;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
            uint32_t t[NV / 2];
#pragma unroll
            for (int e = 0; e < NV / 2; ++e) t[e] = __builtin_amdgcn_perm(v[2 * e + 1][d >> 1], v[2 * e][d >> 1], sel);
            const int dim = 8 * dl + d;
            uint8_t *dst = lds.v[tile & 1][run >> 2][dim >> 4] + chunk_offset(dim & 15, run & 3) + half * 8;
            if constexpr (NV == 8)
                *reinterpret_cast<uint4 *>(dst) = make_uint4(t[0], t[1], t[2], t[3]);
            else
                *reinterpret_cast<uint2 *>(dst) = make_uint2(t[0], t[1]);
        }
    };

    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): of the last item's loads to LDS
    __syncthreads();                     // the tiles' LDS is free
    const int id0 = page_ids(0), id1 = page_ids(1);
    set_places(0, id0);
    set_places(1, id1);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kPartsK; ++n) load_k(0, n);
#pragma unroll
    for (int j = 0; j < NV; ++j) load_v(0, j);

    const int base = chunk_offset(i, g);
    const bool busy = pc.row0 + wave * R * 16 < pc.rows;  // the wave has rows
    half8 qh[R][KS], ql[R][KS];
    float c[R], m[R], l[R];
    int vlo[R], vhi[R], full_lo = 0, full_hi = INT32_MAX;
    float4v o[R][NF];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int mi = pc.row0 + (wave * R + u) * 16 + i;
        const bool live = mi < pc.rows;
        const int i_row = div_group(a, mi), tok = pc.tok0 + i_row, head = pc.kvh * a.group + mi - i_row * a.group;
        c[u] = fmaxf(load_q<KS>(a, a.q + (size_t)tok * a.q_stride + (size_t)head * hd, live, g, qh[u], ql[u]) * score_factor(a),
                     0x1p-126f);
        row_sees(a, sc, need_at, pc, mi, vlo[u], vhi[u]);
        full_lo = max(full_lo, wave_max(vlo[u]));
        full_hi = min(full_hi, wave_min(vhi[u]));
        m[u] = -INFINITY;
        l[u] = 0.0f;
#pragma unroll
        for (int f = 0; f < NF; ++f) o[u][f] = float4v{0, 0, 0, 0};
    }
    store_v(0);

    for (int tile = 0; tile < tiles; ++tile) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): K of this tile is in LDS
        __syncthreads();
        int id2 = -1;
        const uint8_t *kt = lds.k[tile & 1][0][0] + base, *vt = lds.v[tile & 1][0][0] + base;
        // The next tile's loads go out one by one between the products, V's between those with K (it has to be
        // there at the tile's end), K's between those with V: at once they would wait for each other's 16
        // cycles and more of address work.  (Past the last tile: places of none, the first row.)
        auto chunk = [&](int s0, auto loads) {
            constexpr bool kLoads = decltype(loads)::value;
            const int t0 = pc.p0 + tile * T + s0;
            float4v acc[R][NH];
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int h = 0; h < NH; ++h) acc[u][h] = float4v{0, 0, 0, 0};
            // the next kAhead - 1 steps' chunks are on their way from LDS while a step's products run
            constexpr int KG = 2, KN = KS * NH;  // chunks a step, chunks in all: (s, h) = (n / NH, n % NH)
            half8 kk[kAhead][KG];
            auto read_k = [&](int n0) {
#pragma unroll
                for (int e = 0; e < KG; ++e) {
                    const int s = (n0 + e) / NH, h = (n0 + e) % NH;
                    kk[n0 / KG % kAhead][e] = read16(kt + ((s0 / 16 + h) * KS + s) * kChunk);
                }
            };
#pragma unroll
            for (int n = 0; n < (kAhead - 1) * KG && n < KN; n += KG) read_k(n);
#pragma unroll
            for (int n = 0; n < KN; n += KG) {
                if constexpr (kLoads) {
                    constexpr int kEach = (NV * KG + KN - 1) / KN;  // loads a step
#pragma unroll
                    for (int x = 0; x < kEach; ++x)
                        if (n / KG * kEach + x < NV) load_v(tile + 1, n / KG * kEach + x);
                }
                if (n + (kAhead - 1) * KG < KN) read_k(n + (kAhead - 1) * KG);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < R; ++u)
#pragma unroll
                    for (int e = 0; e < KG; ++e)
                        acc[u][(n + e) % NH] = mfma(kk[n / KG % kAhead][e], qh[u][(n + e) / NH], acc[u][(n + e) % NH]);
#pragma unroll
                for (int u = 0; u < R; ++u)
#pragma unroll
                    for (int e = 0; e < KG; ++e)
                        acc[u][(n + e) % NH] = mfma(kk[n / KG % kAhead][e], ql[u][(n + e) / NH], acc[u][(n + e) % NH]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (kLoads) id2 = page_ids(tile + 2);  // after the tile's loads: nothing waits for it alone
            const uint64_t there = __ballot(lane < SP && lds.place[tile % 3][s0 + (lane & (SP - 1))] >= 0);
            const bool edge = t0 < full_lo || t0 + SP > full_hi || there != (SP == 64 ? ~0ull : (1ull << (SP & 63)) - 1);
            uint32_t ph[R][NH][2], pw[R][NH][2];
#pragma unroll
            for (int u = 0; u < R; ++u) {
                float x[4 * NH];
#pragma unroll
                for (int e = 0; e < 4 * NH; ++e) x[e] = acc[u][e >> 2][e & 3];
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 4 * NH; ++e) {
                        const int p = 16 * (e >> 2) + 4 * g + (e & 3), pos = t0 + p;
                        if (pos < vlo[u] || pos >= vhi[u] || !((there >> p) & 1)) x[e] = -INFINITY;
                    }
                }
                float f;
                if (softmax_step<4 * NH>(x, c[u], m[u], l[u], f)) {
#pragma unroll
                    for (int n = 0; n < NF; ++n) o[u][n] *= f;
                }
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) split_p(x[4 * h + 2 * e], x[4 * h + 2 * e + 1], ph[u][h][e], pw[u][h][e]);
            }
#pragma unroll
            for (int b = 0; b < SP / 32; ++b) {
                half8 p_hi[R], p_lo[R];
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    p_hi[u] = as_half8(ph[u][2 * b][0], ph[u][2 * b][1], ph[u][2 * b + 1][0], ph[u][2 * b + 1][1]);
                    p_lo[u] = as_half8(pw[u][2 * b][0], pw[u][2 * b][1], pw[u][2 * b + 1][0], pw[u][2 * b + 1][1]);
                }
                constexpr int VG = 2;  // chunks a step
                half8 vv[kAhead][VG];
                auto read_v = [&](int f0) {
#pragma unroll
                    for (int f = 0; f < VG; ++f)
                        vv[f0 / VG % kAhead][f] = read16(vt + ((s0 / 32 + b) * NF + f0 + f) * kChunk);
                };
#pragma unroll
                for (int f0 = 0; f0 < (kAhead - 1) * VG && f0 < NF; f0 += VG) read_v(f0);
#pragma unroll
                for (int f0 = 0; f0 < NF; f0 += VG) {
                    if constexpr (kLoads) {
                        constexpr int kEach = (kPartsK * VG + NF - 1) / NF;
#pragma unroll
                        for (int x = 0; x < kEach; ++x)
                            if (b == 0 && f0 / VG * kEach + x < kPartsK) load_k(tile + 1, f0 / VG * kEach + x);
                    }
                    if (f0 + (kAhead - 1) * VG < NF) read_v(f0 + (kAhead - 1) * VG);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int u = 0; u < R; ++u)
#pragma unroll
                        for (int f = 0; f < VG; ++f) o[u][f0 + f] = mfma(vv[f0 / VG % kAhead][f], p_hi[u], o[u][f0 + f]);
#pragma unroll
                    for (int u = 0; u < R; ++u)
#pragma unroll
                        for (int f = 0; f < VG; ++f) o[u][f0 + f] = mfma(vv[f0 / VG % kAhead][f], p_lo[u], o[u][f0 + f]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        if (busy) {
            chunk(0, std::true_type{});
#pragma unroll 1
            for (int s0 = SP; s0 < T && pc.p0 + tile * T + s0 < pc.p1; s0 += SP) chunk(s0, std::false_type{});
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) load_v(tile + 1, j);
#pragma unroll
            for (int n = 0; n < kPartsK; ++n) load_k(tile + 1, n);
            id2 = page_ids(tile + 2);
        }
        store_v(tile + 1);
        set_places(tile + 2, id2);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): nothing is on its way to LDS any more
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int mi = pc.row0 + (wave * R + u) * 16 + i;
        const bool live = mi < pc.rows;
        const float lu = row_sum(l[u]);
        float check = lu;
#pragma unroll
        for (int f = 0; f < NF; ++f) check += o[u][f][0] + o[u][f][1] + o[u][f][2] + o[u][f][3];
        check = row_sum(check);
        if (live) {
            const size_t at = part_row(a, pc, to, mi);
            float *dst = to.o + at * hd;
#pragma unroll
            for (int f = 0; f < NF; ++f)
                if (f * 16 < hd)
                    *reinterpret_cast<float4 *>(dst + 16 * f + 4 * g) =
                        make_float4(o[u][f][0], o[u][f][1], o[u][f][2], o[u][f][3]);
            if (g == 0) to.ml[at] = make_float2(m[u] - kShift, usable(check, m[u]) ? lu : kBroken);
        }
    }
}

// ---- the launch --------------------------------------------------------------------

// The prefix's items: of all rows of the batch, in one kind.
struct Shared {
    int rows;           // rows x group
    bool few;           // stream items
    int lo, hi;         // positions any row sees
    int units, items;   // units an item, with its own cost
};

template <int T, int ROWS, int UNIT>
__device__ __forceinline__ Shared shared_work(const PagedAttn &a, const Scan<T> &s, const Totals &t)
{
    Shared p;
    p.rows = uni(s.rs[T] - s.rs[0]) * a.group;
    p.few = !ROWS || p.rows <= kFewRows;
    p.hi = a.prefix_len;
    p.lo = a.window && t.low < INT32_MAX ? min(max(a.prefix_len + t.low - a.window + 1, 0), p.hi) : 0;
    p.items = (p.few ? (p.rows + kRowsA - 1) / kRowsA : (p.rows + ROWS - 1) / (ROWS ? ROWS : 1)) * a.n_kv_heads;
    p.units = p.few ? units_of<kUnitA>(p.lo, p.hi) + kItemCost : units_of<UNIT>(p.lo, p.hi) + block_item_cost(ROWS);
    if (a.prefix_len == 0) p.items = 0;
    return p;
}

// The piece at unit u of the stream or block items, at most `left` units long;
// returns the units taken, the item's index, and whether the piece holds its
// first and last positions.  An item's own cost stands before its first
// unit: a share that ends there has no piece of it (none).
template <bool BLOCK, int T, int ROWS, int UNIT>
__device__ __forceinline__ int find_piece(const PagedAttn &a, const Parts &parts, const Scan<T> &s, const Shared &sh,
                                          int u, int left, Piece &pc, int &item, bool &is_first, bool &is_last,
                                          bool &none)
{
    constexpr int kTile = BLOCK ? ROWS : kRowsA, kStep = BLOCK ? UNIT : kUnitA;
    const int sh_units = sh.few != BLOCK ? sh.items * sh.units : 0;
    int lo, hi, units, within, blk, r = 0;
    pc.pre = u < sh_units;
    if (pc.pre) {
        blk = div_fast(div_fast(u, sh.units, within), a.n_kv_heads, pc.kvh);
        units = sh.units;
        lo = sh.lo;
        hi = sh.hi;
        pc.tok0 = uni(s.rs[0]);
        pc.rows = sh.rows;
        pc.at0 = 0;
        item = (BLOCK ? parts.pre_b : parts.pre_a) + blk * a.n_kv_heads + pc.kvh;
    } else {
        u -= sh_units;
        const int *from = BLOCK ? s.ub : s.ua;
        const int t = share_of<T>(from, u);
        u -= from[t];
        r = t * share<T>(a);
        Request q = request_at(a, s, r);
        if (share<T>(a) > 1) {
            for (;;) {
                int w[2];
                request_units<ROWS, UNIT>(a, q, w[0], w[1]);
                if (u < w[BLOCK] || r + 1 >= a.n_seqs) break;
                u -= w[BLOCK];
                q = request_at(a, s, ++r);
            }
        }
        if constexpr (!BLOCK) {
            own_range(a, q, 0, q.n - 1, lo, hi);
            units = units_of<kUnitA>(lo, hi) + kItemCost;
            blk = div_fast(div_fast(u, units, within), a.n_kv_heads, pc.kvh);
        } else {
            for (blk = 0;; ++blk) {
                tile_range<ROWS>(a, q, blk, lo, hi);
                units = units_of<UNIT>(lo, hi) + block_item_cost(ROWS);
                if (u < units * a.n_kv_heads) break;
                u -= units * a.n_kv_heads;
            }
            pc.kvh = div_fast(u, units, within);
        }
        item = (BLOCK ? parts.own_b : 0) + (q.rs * a.group / kTile + r + blk) * a.n_kv_heads + pc.kvh;
        pc.tok0 = uni(q.rs);
        pc.rows = uni(q.n * a.group);
        pc.at0 = uni(q.len - q.n);
    }
    units = uni(units);
    within = uni(within);
    const int take = min(units - within, left), cost = BLOCK ? block_item_cost(ROWS) : kItemCost;
    const int from = max(within - cost, 0), to = max(within + take - cost, 0);
    item = uni(item);
    pc.table = pc.pre ? a.prefix : a.table + (size_t)uni(r) * a.table_stride;
    pc.kvh = uni(pc.kvh);
    pc.row0 = uni(blk) * kTile;
    pc.p0 = uni(lo) + from * kStep;
    pc.p1 = min(uni(hi), uni(lo) + to * kStep);
    is_first = from == 0;
    is_last = within + take == units;
    none = to == from;
    return take;
}

template <int DP, int KF, int VF>
struct KernelLds {
    Scan<64 * waves_of(DP, KF, VF)> scan;
    WaveLds<DP, KF, VF> wave[waves_of(DP, KF, VF)];
};
template <int DP>
struct KernelLds<DP, 0, 0> {
    Scan<64 * waves_of(DP, 0, 0)> scan;
    union {
        WaveLds<DP, 0, 0> wave[waves_of(DP, 0, 0)];
        BlockLds<DP> block;
    };
};

// Quantised caches have stream items alone.  ONCE: K and V of stream items are
// loaded with the non-temporal hint, which pays where the requests' own positions are all there is
// (256 x 1000 positions of 4 heads of 256 dims: 212 us against 223; 4 x 32000 of 8 heads of 128: 107
// against 116) and not beside a prefix's blocks (256 requests of 300 positions behind 8192: 225 us against 218).
// At most two row tiles read the same rows of an f16 cache so; of a quantised one all do.
template <int DP, int KF, int VF, bool ONCE>
__global__ __launch_bounds__(64 * waves_of(DP, KF, VF)) void paged_attn_kernel(PagedAttn a, Parts parts)
{
    constexpr bool kBlocks = !KF && !VF;
    constexpr int kWaves = waves_of(DP, KF, VF), T = 64 * kWaves;
    constexpr int kUnitB = unit_b(DP), kRowsB = kBlocks ? rows_b(DP) : 0;
    __shared__ KernelLds<DP, KF, VF> lds;
    const Scan<T> &s = lds.scan;
    const int wg = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Totals totals = scan_requests<T, kRowsB, kUnitB>(a, lds.scan);
    // row starts that do not ascend: nothing is computed
    if (wg == 0 && tid == 0) {
        *reinterpret_cast<int4 *>(parts.head) = make_int4(totals.ok, s.rs[0], s.rs[T], 0);
        if (!totals.ok) page_fault(a.faults);
    }
    if (!totals.ok) return;
    const Shared sh = shared_work<T, kRowsB, kUnitB>(a, s, totals);
    const int sh_units = sh.items * sh.units;
    const int ua = uni(s.ua[T]) + (sh.few ? sh_units : 0), ub = uni(s.ub[T]) + (sh.few ? 0 : sh_units);

    // the request of each row, for joining the parts
    for (int row = s.rs[0] + wg * T + tid; row < s.rs[T]; row += parts.wgs * T) {
        const int r = request_of(a, s, row);
        const Request q = request_at(a, s, r);
        parts.row_item[row] = make_int4(r, q.rs, q.n, 0);
    }

    int wb = 0;
    if (kBlocks && ub > 0) {
        wb = parts.wgs;
        if (ua > 0) {
            const float fb = (float)ub * (kBlockCost * kWaves * kRowsB / 32), fa = (float)ua;
            wb = min(max((int)(parts.wgs * fb / (fa + fb) + 0.5f), 1), parts.wgs - 1);
        }
    }
    Piece pc;
    int item;
    bool first, last, none;
    if constexpr (kBlocks) {
        if (wg < wb) {
            int rest;
            const int quota = uni(div_fast(ub + wb - 1, wb, rest)), end = min(ub, (wg + 1) * quota);
            for (int u = wg * quota; u < end;) {
                u += find_piece<true, T, kRowsB, kUnitB>(a, parts, s, sh, u, end - u, pc, item, first, last, none);
                if (none) continue;
                const size_t row = (size_t)wg * kRowsB;
                const Dest to = first ? Dest{parts.o[!pc.pre], parts.ml[!pc.pre], true}
                                      : Dest{parts.o_b + row * a.head_dim, parts.ml_b + row, false};
                if (tid == 0 && first) parts.first[item] = wg;
                if (tid == 0 && last) parts.last[item] = wg;
                block_item<DP>(a, s, totals.need_at, pc, lds.block, to);
            }
            return;
        }
    }
    const int worker = (wg - wb) + (parts.wgs - wb) * wave, workers = (parts.wgs - wb) * kWaves;
    int rest;
    const int quota = uni(div_fast(ua + workers - 1, workers, rest)), end = min(ua, (worker + 1) * quota);
    for (int u = worker * quota; u < end;) {
        u += find_piece<false, T, kRowsB, kUnitB>(a, parts, s, sh, u, end - u, pc, item, first, last, none);
        if (none) continue;
        const size_t row = (size_t)worker * kRowsA;
        const Dest to = first ? Dest{parts.o[!pc.pre], parts.ml[!pc.pre], true}
                              : Dest{parts.o_a + row * a.head_dim, parts.ml_a + row, false};
        if ((tid & 63) == 0 && first) parts.first[item] = worker;
        if ((tid & 63) == 0 && last) parts.last[item] = worker;
        stream_item<DP, KF, VF, ONCE>(a, s, totals.need_at, pc, lds.wave[wave], to);
    }
}

// ---- joining the parts ---------------------------------------------------------------

// The f16 terms of p and q turn an infinite value into NaN, and a weight of 0
// times an infinity that its row does not see is one too; and scores beyond
// kFarScore leave p's range.  So a row with a part that is not usable is formed again here, one position after the
// other in f32 (`waves` waves taking turns, q and o in LDS); a program whose values are finite and whose scores
// are below 7e5 never gets here.
__device__ __forceinline__ void slow_row(const PagedAttn &a, int row, int r, int h, int wave, int waves, float *s_q,
                                         float *s_o, float &m, float &l)
{
    const int lane = threadIdx.x & 63, hd = a.head_dim, kvh = div_group(a, h);
    const int len = clamp_len(a, a.lens[r]), at = a.prefix_len + len - (a.row_start[r + 1] - row);
    const int first = a.window ? max(0, at - a.window + 1) : 0;
    const HeadRows k_rows = head_rows(a, a.k, a.k_fmt, kvh), v_rows = head_rows(a, a.v, a.v_fmt, kvh);
#pragma unroll 1
    for (int d0 = 0; d0 < hd; d0 += 64) {
        const int d = d0 + lane;
        const float x = d < hd ? a.q[(size_t)row * a.q_stride + (size_t)h * hd + d] : 0.0f;
        uint32_t db;
        int sum;
        const float q8 = (float)q8_0_block32(x, db, sum) * f16_bits_to_f32(db);  // blocks of 32 dims, a half wave each
        if (d < hd) {
            s_q[d] = a.k_fmt == 0 ? x : q8;
            s_o[d] = 0.0f;
        }
    }
    m = -INFINITY;
    l = 0.0f;
#pragma unroll 1
    for (int t = first + wave; t <= at; t += waves) {
        const bool pre = t < a.prefix_len;
        const int place = pre ? place_at(a, a.prefix, t) : place_at(a, a.table + (size_t)r * a.table_stride, t - a.prefix_len);
        if (place < 0) continue;
        const uint8_t *kr = k_rows.row(place), *vr = v_rows.row(place);
        float s = 0.0f;
#pragma unroll 1
        for (int d = lane; d < hd; d += 64) s = fmaf(s_q[d], kv_value(kr, a.k_fmt, d), s);
        for (int y = 32; y; y >>= 1) s += __shfl_xor(s, y, 64);
        s *= a.scale * kLog2e;
        if (s == -INFINITY) continue;  // no weight
        const float m2 = fmaxf(m, s), f = exp2f(m - m2), w = exp2f(s - m2);
        l = l * f + w;
#pragma unroll 1
        for (int d = lane; d < hd; d += 64) s_o[d] = s_o[d] * f + w * kv_value(vr, a.v_fmt, d);
        m = m2;
    }
}

// What a row without any weight gives: 0 if no position that it sees has a place, else 0 / 0, since all its scores
// were -inf.  64 positions a step, since a table that leads nowhere has them all looked at.
__device__ __forceinline__ float without_weight(const PagedAttn &a, int row, int r)
{
    const int len = clamp_len(a, a.lens[r]), at = a.prefix_len + len - (a.row_start[r + 1] - row);
#pragma unroll 1
    for (int t0 = a.window ? max(0, at - a.window + 1) : 0; t0 <= at; t0 += 64) {
        const int t = t0 + (threadIdx.x & 63);
        const int32_t *table = t < a.prefix_len ? a.prefix : a.table + (size_t)r * a.table_stride;
        if (__any(t <= at && place_at(a, table, t < a.prefix_len ? t : t - a.prefix_len) >= 0)) return NAN;
    }
    return 0.0f;
}

// Joins the parts of each row and head.  W waves share a row and head, lane groups
// take a part each, a lane four dims of it, with a running maximum of their own; lane groups and waves
// join as parts do.  Two round trips after the row's request: where the parts are, then the parts.  Bound by them
// (5.5 us for 8 pairs, 7 for 256 in some ten parts) or by the parts' bytes (17 us for 2134 rows of 8 heads of 256 dims: 54 MB).
template <int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void paged_merge_kernel(PagedAttn a, Parts parts)
{
    constexpr int kAhead = 3, kWaves = W == 1 ? 4 : W;
    __shared__ float s_o[kWaves][512], s_q[kWaves][512], s_l[kWaves], s_m[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), hd = a.head_dim;
    const int pair = blockIdx.x * (kWaves / W) + wave / W, row = pair / a.n_heads, h = pair - row * a.n_heads;
    if (row >= a.max_rows) return;  // W == 1: the last workgroup's spare waves (no barrier there)
    const int4 head = *reinterpret_cast<const int4 *>(parts.head);
    const int4 ri = parts.row_item[row];
    if (!head.x || row < head.y || row >= head.z) return;  // W > 1: the whole workgroup
    const int kvh = div_group(a, h), gq = h - kvh * a.group;
    const size_t base = (size_t)row * a.n_heads + h;
    // the two items of the row: the prefix's, its own
    int w0[2], n[2], at[2], rows[2], item[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int row0 = x ? ri.y : head.y, m = (x ? ri.z : head.z - head.y) * a.group, mi = (row - row0) * a.group + gq;
        const bool block = parts.rows_b && m > kFewRows;
        rows[x] = block ? parts.rows_b : kRowsA;
        const int sh = __builtin_ctz(rows[x]), tile = mi >> sh;
        at[x] = mi - (tile << sh);
        const int at0 = x ? (block ? parts.own_b : 0) : (block ? parts.pre_b : parts.pre_a);
        item[x] = at0 + ((x ? (ri.y * a.group >> sh) + ri.x : 0) + tile) * a.n_kv_heads + kvh;
    }
    w0[0] = a.prefix_len > 0 ? parts.first[item[0]] : 0;
    w0[1] = parts.first[item[1]];
    n[0] = a.prefix_len > 0 ? parts.last[item[0]] - w0[0] + 1 : 0;
    n[1] = parts.last[item[1]] - w0[1] + 1;
    const int total = n[0] + n[1];
    auto part = [&](int k, const float *&po, const float2 *&pml) {
        const int x = k >= n[0], j = k - (x ? n[0] : 0);
        const bool block = rows[x] != kRowsA;
        const size_t r = (size_t)(w0[x] + j) * rows[x] + at[x];
        po = j == 0 ? parts.o[x] + base * hd : (block ? parts.o_b : parts.o_a) + r * hd;
        pml = j == 0 ? parts.ml[x] + base : (block ? parts.ml_b : parts.ml_a) + r;
    };
    // lanes over dims (four each; heads beyond 256 dims in two turns), lane groups over parts
    const int lanes = hd <= 32 ? 8 : hd <= 64 ? 16 : hd <= 128 ? 32 : 64, groups = 64 / lanes * W;
    const int sub = (wave % W) * (64 / lanes) + lane / lanes, d0 = (lane % lanes) * 4;
    bool broken = false;
    float4 o[2] = {};
    float m = -INFINITY, l = 0.0f;
    for (int k0 = sub; k0 < total; k0 += groups * kAhead) {
        float4 v[kAhead][2];
        float2 ml[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const float *po;
            const float2 *pml;
            const int k = k0 + e * groups;
            part(min(k, total - 1), po, pml);
            ml[e] = k < total ? *pml : make_float2(0.0f, 0.0f);
            v[e][0] = d0 < hd ? *reinterpret_cast<const float4 *>(po + d0) : make_float4(0, 0, 0, 0);
            v[e][1] = d0 + 256 < hd ? *reinterpret_cast<const float4 *>(po + d0 + 256) : make_float4(0, 0, 0, 0);
        }
        float m2 = m;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            broken |= ml[e].y < 0.0f;
            if (ml[e].y != 0.0f) m2 = fmaxf(m2, ml[e].x);
        }
        if (m2 == -INFINITY) continue;  // nothing seen so far
        const float f = exp2_hw(m - m2);
        m = m2;
        l *= f;
#pragma unroll
        for (int x = 0; x < 2; ++x) o[x] = make_float4(o[x].x * f, o[x].y * f, o[x].z * f, o[x].w * f);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (ml[e].y == 0.0f) continue;  // saw nothing
            const float w = exp2_hw(ml[e].x - m);
            l += ml[e].y * w;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                o[x].x += v[e][x].x * w;
                o[x].y += v[e][x].y * w;
                o[x].z += v[e][x].z * w;
                o[x].w += v[e][x].w * w;
            }
        }
    }
    broken = __any(broken);
    if (lanes < 64) {
        float m2 = m;
        for (int x = lanes; x < 64; x <<= 1) m2 = fmaxf(m2, __shfl_xor(m2, x, 64));
        const float f = m == -INFINITY ? 0.0f : exp2_hw(m - m2);
        m = m2;
        l *= f;
        o[0] = make_float4(o[0].x * f, o[0].y * f, o[0].z * f, o[0].w * f);  // o[1]: past 256 dims alone
        for (int x = lanes; x < 64; x <<= 1) {
            l += __shfl_xor(l, x, 64);
            o[0].x += __shfl_xor(o[0].x, x, 64);
            o[0].y += __shfl_xor(o[0].y, x, 64);
            o[0].z += __shfl_xor(o[0].z, x, 64);
            o[0].w += __shfl_xor(o[0].w, x, 64);
        }
    }
    if constexpr (W == 1) {
        if (broken) slow_row(a, row, ri.x, h, 0, 1, s_q[wave], s_o[wave], m, l);
        const float none = l == 0.0f ? without_weight(a, row, ri.x) : 0.0f;
        if (broken) {
            for (int d = lane; d < hd; d += 64) a.out[base * hd + d] = l == 0.0f ? none : s_o[wave][d] / l;
            return;
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int d = d0 + 256 * y;
            if (lane < lanes && d < hd)
                *reinterpret_cast<float4 *>(a.out + base * hd + d) =
                    l == 0.0f ? make_float4(none, none, none, none) : make_float4(o[y].x / l, o[y].y / l, o[y].z / l, o[y].w / l);
        }
    } else {
        if (lane < lanes) {
            if (d0 < hd) *reinterpret_cast<float4 *>(&s_o[wave][d0]) = o[0];
            if (d0 + 256 < hd) *reinterpret_cast<float4 *>(&s_o[wave][d0 + 256]) = o[1];
        }
        if (lane == 0) {
            s_m[wave] = m;
            s_l[wave] = l;
        }
        if (__syncthreads_or(broken)) {
            slow_row(a, row, ri.x, h, wave, W, s_q[wave], s_o[wave], m, l);
            if (lane == 0) {
                s_m[wave] = m;
                s_l[wave] = l;
            }
            __syncthreads();
        }
        float most = s_m[0], sum = 0.0f, f[W];
#pragma unroll
        for (int w = 1; w < W; ++w) most = fmaxf(most, s_m[w]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            f[w] = s_l[w] == 0.0f ? 0.0f : s_l[w] != s_l[w] ? s_l[w] : exp2_hw(s_m[w] - most);  // NaN stays
            sum += f[w] == 0.0f ? 0.0f : s_l[w] * f[w];
        }
        const float none = sum == 0.0f ? without_weight(a, row, ri.x) : 0.0f;
        for (int d = tid; d < hd; d += 64 * W) {
            float x = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) x += f[w] == 0.0f ? 0.0f : s_o[w][d] * f[w];
            a.out[base * hd + d] = sum == 0.0f ? none : x / sum;
        }
    }
}

int padded_dim(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : head_dim <= 256 ? 256 : 512; }

Parts layout(const PagedAttn &a, uint8_t *base, size_t &bytes)
{
    Parts p{};
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t *x = base + at;
        at += align_up(n, 256);
        return x;
    };
    const bool quant = a.k_fmt != 0 || a.v_fmt != 0;
    const int dp = padded_dim(a.head_dim);
    p.wgs = 256;  // one a CU: they hold most of its registers or LDS
    p.waves = waves_of(dp, a.k_fmt, a.v_fmt);
    p.rows_b = quant ? 0 : rows_b(dp);
    const size_t heads = (size_t)a.max_rows * a.n_heads, hd = a.head_dim;
    const size_t group_rows = (size_t)a.max_rows * a.group;
    const size_t tiles_a = group_rows / kRowsA + 1, tiles_b = p.rows_b ? group_rows / p.rows_b + 1 : 0, kv = a.n_kv_heads;
    p.pre_a = (int)((tiles_a + a.n_seqs) * kv);
    p.own_b = (int)(p.pre_a + tiles_a * kv);
    p.pre_b = (int)(p.own_b + (p.rows_b ? tiles_b + a.n_seqs : 0) * kv);
    const size_t items = p.pre_b + tiles_b * kv;
    for (int k = 0; k < 2; ++k) {
        const bool used = k == 1 || a.prefix_len > 0;
        p.o[k] = reinterpret_cast<float *>(take(used ? heads * hd * 4 : 0));
        p.ml[k] = reinterpret_cast<float2 *>(take(used ? heads * 8 : 0));
    }
    const size_t workers = (size_t)p.wgs * p.waves, wg_rows = (size_t)p.wgs * p.rows_b;
    p.o_a = reinterpret_cast<float *>(take(workers * kRowsA * hd * 4));
    p.ml_a = reinterpret_cast<float2 *>(take(workers * kRowsA * 8));
    p.o_b = reinterpret_cast<float *>(take(wg_rows * hd * 4));
    p.ml_b = reinterpret_cast<float2 *>(take(wg_rows * 8));
    p.first = reinterpret_cast<int32_t *>(take(items * 4));
    p.last = reinterpret_cast<int32_t *>(take(items * 4));
    p.row_item = reinterpret_cast<int4 *>(take((size_t)a.max_rows * 16));
    p.head = reinterpret_cast<int32_t *>(take(16));
    bytes = at;
    return p;
}

template <int DP>
void launch_dp(mrml_hip_ctx *ctx, const PagedAttn &a, const Parts &p)
{
    const dim3 grid(p.wgs), block(64 * p.waves);
#define MRML_PAGED_CASE(KF, VF)                                                                                       \
    case 3 * KF + VF:                                                                                                 \
        hipLaunchKernelGGL((paged_attn_kernel<DP, KF, VF, false>), grid, block, 0, ctx->stream, a, p);               \
        break;
    switch (3 * a.k_fmt + a.v_fmt) {
        MRML_PAGED_CASE(0, 1)
        MRML_PAGED_CASE(0, 2)
        MRML_PAGED_CASE(1, 0)
        MRML_PAGED_CASE(1, 1)
        MRML_PAGED_CASE(1, 2)
        MRML_PAGED_CASE(2, 0)
        MRML_PAGED_CASE(2, 1)
        MRML_PAGED_CASE(2, 2)
    default:
        if (a.prefix_len == 0)
            hipLaunchKernelGGL((paged_attn_kernel<DP, 0, 0, true>), grid, block, 0, ctx->stream, a, p);
        else
            hipLaunchKernelGGL((paged_attn_kernel<DP, 0, 0, false>), grid, block, 0, ctx->stream, a, p);
    }
#undef MRML_PAGED_CASE
}

}  // namespace

// Stream units: at most two row tiles a request where there are block items, else tiles of 16 of all rows, over
// the longest table row; and the prefix's.  Block units are fewer than half of what their rows would give in tiles
// of 16 (64 rows of 32 positions, at least).  Rows times heads have to fit an int too.
bool paged_attn_countable(const PagedAttn &a)
{
    const double kv = a.n_kv_heads, rows = (double)a.max_rows * a.group, seqs = std::min(a.n_seqs, a.max_rows);
    const bool quant = a.k_fmt != 0 || a.v_fmt != 0;
    const double tiles = rows / kRowsA + seqs, own = a.longest / kUnitA + 1 + kItemCost, pre = a.prefix_len / kUnitA + 1 + kItemCost;
    const double a_units = quant ? tiles * (own + pre) : 2 * seqs * own + 2 * pre;
    const double b_units = quant ? 0 : tiles / 2 * (own + pre + 16);  // 16: two block items' own costs at most
    const double most = 1 << 30;
    return kv * (a_units + b_units) < most && kv * (2 * tiles + 2.0 * a.n_seqs + 8) < most && (double)a.max_rows * a.n_heads < most;
}

size_t paged_attn_scratch_bytes(const PagedAttn &a)
{
    size_t bytes;
    layout(a, nullptr, bytes);
    return bytes;
}

int launch_paged_attn(mrml_hip_ctx *ctx, const PagedAttn &a, void *scratch)
{
    size_t bytes;
    const Parts p = layout(a, reinterpret_cast<uint8_t *>(scratch), bytes);
    switch (padded_dim(a.head_dim)) {
    case 64: launch_dp<64>(ctx, a, p); break;
    case 128: launch_dp<128>(ctx, a, p); break;
    case 256: launch_dp<256>(ctx, a, p); break;
    default: launch_dp<512>(ctx, a, p); break;
    }
    if (int rc = check_launch(ctx, "paged_attn_kernel")) return rc;
    // Waves a row and head by how many there can be; how many there are is on the device (32 requests of 8 heads with
    // max_rows 256 or more get one wave a pair: 39 us a call, 30 with max_rows 32).  Measured on both sides of the
    // lines (us): 32 pairs in 500 parts each 86 with 4 and 60 with 16 (the whole call), 256 pairs 7.1 and 6.8, 408 pairs
    // 7.2 and 9.0, 732 pairs 5.3 and 10.8; 408 pairs 16.2 with one and 7.4 with 4, 732 8.4 and 5.6, 2048 11.9 and
    // 13.7, 4096 5.2 and 12.0.
    const int pairs = a.max_rows * a.n_heads;
    if (pairs > 1024)
        hipLaunchKernelGGL(paged_merge_kernel<1>, dim3((pairs + 3) / 4), dim3(256), 0, ctx->stream, a, p);
    else if (pairs > 256)
        hipLaunchKernelGGL(paged_merge_kernel<4>, dim3(pairs), dim3(256), 0, ctx->stream, a, p);
    else
        hipLaunchKernelGGL(paged_merge_kernel<16>, dim3(pairs), dim3(1024), 0, ctx->stream, a, p);
    return check_launch(ctx, "paged_merge_kernel");
}

}  // namespace mrml
