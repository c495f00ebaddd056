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
// of items -- (16 or 128 query rows that share their K and V) x (a kv head) x
// (a range of positions of the prefix or of one request) -- cut into units of
// positions and dealt out evenly; paged_merge_kernel joins the parts.
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
constexpr int kScanT = 256;       // threads of a workgroup
constexpr int kRowsA = 16, kUnitA = 32;  // rows and positions of a stream item's tile (one wave)
constexpr int kRowsB = 128;              // rows of a block item's tile (four waves)
constexpr int kFewRows = 32;             // groups of at most so many rows are stream items
// Relative cost of a unit on one workgroup, for the split of the workgroups:
// a block unit keeps the MFMA of all four waves busy, four stream units run side by side.
constexpr int kCostA = 1, kCostB = 8;

constexpr int unit_b(int dp) { return 16384 / dp; }

// Device scratch of a call (paged_attn_scratch_bytes).
struct Parts {
    float *o[2];         // first part of each row's prefix and own item: [row][head][head_dim]
    float2 *ml[2];       // (m, l) of those
    float *o_a, *o_b;    // later parts, by worker: [worker][16][head_dim], [workgroup][128][head_dim]
    float2 *ml_a, *ml_b;
    int32_t *first, *last;  // workers that hold an item's first and last unit
    int2 *row_item;         // {the own items' first index, row within the request}, type in bit 30 of y
    int32_t *head;          // {rows are sound, first row, rows}
    int items_a;            // index of the first block item
    int wgs;
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

struct Scan {  // per thread's share of the requests: exclusive sums, in LDS
    int ua[kScanT + 1], ub[kScanT + 1];  // units
    int ia[kScanT + 1], ib[kScanT + 1];  // items
    int rs[kScanT + 1];                  // first row
    int sum[8][4];
    int bad, low, need_at;
    float size;
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

__device__ __forceinline__ const uint8_t *kv_row(const PagedAttn &a, const uint8_t *cache, int row_bytes, int place,
                                                 int kvh)
{
    return cache + ((size_t)(uint32_t)max(place, 0) * a.n_kv_heads + kvh) * row_bytes;
}

// ---- the requests' shares of the work --------------------------------------------

struct Request {
    int rs, n, len;  // first row, rows, own length (within its table row)
};

__device__ __forceinline__ Request request_at(const PagedAttn &a, int r)
{
    Request q;
    q.rs = a.row_start[r];
    q.n = a.row_start[r + 1] - q.rs;
    q.len = min(max(a.lens[r], 0), a.table_stride * a.map.page_size);
    return q;
}

// Own positions that rows i0..i1 of a request see: [lo, hi).
__device__ __forceinline__ void own_range(const PagedAttn &a, const Request &q, int i0, int i1, int &lo, int &hi)
{
    hi = max(q.len - q.n + i1 + 1, 0);
    lo = a.window ? min(max(q.len - q.n + i0 - a.window + 1, 0), hi) : 0;
}

__device__ __forceinline__ int units_of(int lo, int hi, int unit) { return max(1, (hi - lo + unit - 1) / unit); }

__device__ __forceinline__ int own_units_a(const PagedAttn &a, const Request &q)
{
    int lo, hi;
    own_range(a, q, 0, q.n - 1, lo, hi);
    return units_of(lo, hi, kUnitA);
}

__device__ __forceinline__ int own_units_b(const PagedAttn &a, const Request &q, int block, int unit)
{
    int lo, hi;
    const int last = min(q.n * a.group, (block + 1) * kRowsB) - 1;
    own_range(a, q, block * kRowsB / a.group, last / a.group, lo, hi);
    return units_of(lo, hi, unit);
}

// {stream units, block units, stream items, block items} of a request; returns the units as a float, which cannot
// overflow.
__device__ __forceinline__ float request_work(const PagedAttn &a, const Request &q, bool blocks, int unit, int w[4])
{
    w[0] = w[1] = w[2] = w[3] = 0;
    if (q.n <= 0) return 0.0f;
    const int m = q.n * a.group;
    if (!blocks || m <= kFewRows) {
        w[2] = (m + kRowsA - 1) / kRowsA * a.n_kv_heads;
        w[0] = w[2] * own_units_a(a, q);
        return (float)w[2] * (float)own_units_a(a, q);
    } else {
        const int nb = (m + kRowsB - 1) / kRowsB;
        float size = 0.0f;
        for (int b = 0; b < nb; ++b) {
            const int n = own_units_b(a, q, b, unit);
            w[1] += n;
            size += (float)n;
        }
        w[1] *= a.n_kv_heads;
        w[3] = nb * a.n_kv_heads;
        return size * (float)a.n_kv_heads;
    }
}

// Every workgroup forms the same sums over all requests (a few loads a thread).
__device__ void scan_requests(const PagedAttn &a, Scan &s, bool blocks, int unit)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.n_seqs + kScanT - 1) / kScanT, r0 = tid * per;
    if (tid == 0) {
        s.bad = 0;
        s.low = INT32_MAX;
        s.need_at = 0;
        s.size = 0.0f;
    }
    int w[4] = {0, 0, 0, 0}, bad = 0, low = INT32_MAX, neg = 0;
    for (int r = r0; r < min(r0 + per, a.n_seqs); ++r) {
        const int rs = a.row_start[r], re = a.row_start[r + 1];
        bad |= rs < 0 || re < rs || re > a.max_rows;
        if (blockIdx.x == 0 && (uint32_t)a.lens[r] > (uint32_t)(a.table_stride * a.map.page_size)) page_fault(a.faults);
    }
    __syncthreads();
    if (bad) s.bad = 1;
    __syncthreads();
    if (s.bad) return;
    float size = 0.0f;
    for (int r = r0; r < min(r0 + per, a.n_seqs); ++r) {
        const Request q = request_at(a, r);
        int x[4];
        size += request_work(a, q, blocks, unit, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] += x[k];
        if (q.n > 0) {
            low = min(low, q.len - q.n);
            neg |= q.len < q.n;
        }
    }
    s.rs[tid] = a.row_start[min(r0, a.n_seqs)];
    if (tid == 0) s.rs[kScanT] = a.row_start[a.n_seqs];
    if (low < INT32_MAX) atomicMin(&s.low, low);
    if (neg) s.need_at = 1;
    if (size > 0.0f) atomicAdd(&s.size, size);  // a rough figure, compared with one bound
    int inc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        int x = w[k];
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(x, d, 64);
            if (lane >= d) x += y;
        }
        inc[k] = x;
        if (lane == 63) s.sum[wave][k] = x;
    }
    __syncthreads();
    int *dst[4] = {s.ua, s.ub, s.ia, s.ib};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        int before = 0;
        for (int v = 0; v < wave; ++v) before += s.sum[v][k];
        dst[k][tid] = before + inc[k] - w[k];
        if (tid == kScanT - 1) dst[k][kScanT] = before + inc[k];
    }
    __syncthreads();
}

// The thread whose share [from[t], from[t + 1]) holds x (from ascending, from[0] <= x < from[256]).
__device__ __forceinline__ int share_of(const int *from, int x)
{
    int lo = 0, hi = kScanT - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (from[mid] <= x)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// The request of a row (the last one that starts at or before it and has rows).
__device__ __forceinline__ int request_of(const PagedAttn &a, const Scan &s, int row)
{
    const int per = (a.n_seqs + kScanT - 1) / kScanT;
    int r = share_of(s.rs, row) * per;
    while (r + 1 < a.n_seqs && a.row_start[r + 1] <= row) ++r;
    return r;
}

// ---- a row on its own -------------------------------------------------------------
//
// The f16 terms of p and q turn an infinite value into NaN, and a weight of 0
// times an infinity that its row does not see is one too.  So a row whose part
// came out NaN is formed again, one position after the other in f32, by the
// wave; a program whose values are finite never gets here.
__device__ __noinline__ void slow_row(const PagedAttn &a, const Piece &pc, int mi, int vlo, int vhi, float *o_dst,
                                      float2 *ml_dst)
{
    constexpr int E = 8;  // values a lane at most
    const int lane = threadIdx.x & 63, hd = a.head_dim;
    const int tok = pc.tok0 + mi / a.group, head = pc.kvh * a.group + mi % a.group;
    const float *qr = a.q + (size_t)tok * a.q_stride + (size_t)head * hd;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = e * 64 + lane;
        const float x = d < hd ? qr[d] : 0.0f;
        q[e] = x;
        o[e] = 0.0f;
        if (a.k_fmt != 0) {
            uint32_t db;
            int qs;
            q[e] = (float)q8_0_block32(x, db, qs) * f16_bits_to_f32(db);
        }
    }
    const int kb = kv_row_bytes(a.k_fmt, hd), vb = kv_row_bytes(a.v_fmt, hd);
    for (int t = max(pc.p0, vlo); t < min(pc.p1, vhi); ++t) {
        const int place = place_at(a, pc.table, t);
        if (place < 0) continue;
        const uint8_t *kr = kv_row(a, a.k, kb, place, pc.kvh), *vr = kv_row(a, a.v, vb, place, pc.kvh);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e * 64 + lane < hd) s = fmaf(q[e], kv_value(kr, a.k_fmt, e * 64 + lane), s);
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x, 64);
        s *= a.scale * kLog2e;
        if (s == -INFINITY) continue;  // no weight
        const float m2 = fmaxf(m, s), f = exp2f(m - m2), w = exp2f(s - m2);
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e * 64 + lane < hd) o[e] = o[e] * f + w * kv_value(vr, a.v_fmt, e * 64 + lane);
        m = m2;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e * 64 + lane < hd) o_dst[e * 64 + lane] = o[e];
    if (lane == 0) *ml_dst = make_float2(m, l);
}

// ---- query rows ------------------------------------------------------------------

__device__ __forceinline__ size_t part_row(const PagedAttn &a, const Piece &pc, const Dest &d, int mi)
{
    return d.own ? (size_t)(pc.tok0 + mi / a.group) * a.n_heads + pc.kvh * a.group + mi % a.group : (size_t)(mi - pc.row0);
}

// What row mi of a piece's group sees, in the source's positions: [vlo, vhi).
__device__ __forceinline__ void row_sees(const PagedAttn &a, const Scan &s, const Piece &pc, int mi, int &vlo, int &vhi)
{
    vlo = 0;
    vhi = INT32_MAX;
    if (mi >= pc.rows) return;
    const int tok = pc.tok0 + mi / a.group;
    if (!pc.pre) {
        const int at = pc.at0 + mi / a.group;
        vhi = at + 1;
        vlo = a.window ? at - a.window + 1 : 0;
    } else if (s.need_at || a.window) {
        const Request q = request_at(a, request_of(a, s, tok));
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

// q of one row as two f16 terms of q * 2^k, lane group g holding dims 32 s + 8 g ..: 
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
    const float up = as_f((uint32_t)(267 - ex) << 23);
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
    const float rx = x - (float)h[0], ry = y - (float)h[1];
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

// Running softmax of one row: x holds N scores of this lane (log2 domain, -inf
// where masked), which become p * 2^14; m and l are brought up to date, true if
// o has to be multiplied by f.
template <int N>
__device__ __forceinline__ bool softmax_step(float *x, float &m, float &l, float &f)
{
    float top = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
    top = row_max(top);
    const bool grow = top > m + kSlack;
    f = 1.0f;
    const bool any = __any(grow);
    if (any) {
        const float m2 = grow ? top : m;
        f = grow ? exp2_hw(m - m2) : 1.0f;  // 0 from -inf
        l *= f;
        m = m2;
    }
    const float base = m == -INFINITY ? 0.0f : m - kShift;
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        x[e] = exp2_hw(x[e] - base);
        sum += x[e];
    }
    l += sum;
    return any;
}

// ---- stream items: a wave, 16 query rows, K and V straight from memory ------------
//
// Per tile of 32 positions a lane loads K of position lane % 16 (+ 16) in 16-byte
// pieces, which are the product's operand as they are, and V of 8 positions in
// 16-byte pieces of 8 dims.  V's operand wants 8 positions of one dim: an 8 x 8
// transpose inside the lane's registers, one v_perm a pair; the dims then lie
// 8 apart over the operand's rows, which only the store of o has to know.  With
// K of the next tile and V of this one in flight a wave keeps 32 KB on the
// way (head_dim 256), so one wave a SIMD suffices to be bound by HBM.
//
// Quantised K is multiplied as the ring attention does it: q as Q8_0 blocks,
// each block's integer sum on the int8 MFMA (16x16x32: one block a
// step), times both scales in f32.  There q is the left operand, so that a
// lane's position, and K's scale with it, is fixed; the tile of scores changes
// sides through LDS once.  Quantised V enters as f16 terms too: d * q has at most
// 19 bits, hi = its rounding, lo = fma(d, q, -hi), both exact.

struct __attribute__((packed, aligned(2))) Bytes8 {
    uint32_t a, b;
};

constexpr int kTrRow = 36;  // floats a query row of the score tile in LDS

struct WaveLds {
    int place[32];
    float scores[16 * kTrRow];
};

// Query rows for a quantised K: operand bytes, and scale and sum of each block
// for the four rows that this lane's results belong to.
template <int KS>
struct QuantQ {
    long q[KS];
    float4v d[KS];
    int4v sum8[KS];  // -8 * sum of the block's quants: what Q4_0's offset takes away
};

template <int KS>
__device__ __forceinline__ void load_quant_q(const PagedAttn &a, const float *row, bool live, int g, QuantQ<KS> &out)
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
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            out.d[s][r] = __shfl(d, 4 * g + r, 64);
            out.sum8[s][r] = a.k_fmt == 2 ? -8 * __shfl(sum, 4 * g + r, 64) : 0;
        }
    }
}

template <int DP, bool KQ, bool VQ>
__device__ __forceinline__ void stream_item(const PagedAttn &a, const Scan &sc, const Piece &pc, WaveLds &lds,
                                            const Dest &to)
{
    constexpr int KS = DP / 32, NG = DP < 128 ? 1 : DP / 128;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, hd = a.head_dim;
    const int mi = pc.row0 + i;
    const bool live = mi < pc.rows;
    const int tok = pc.tok0 + mi / a.group, head = pc.kvh * a.group + mi % a.group;
    const float *q_row = a.q + (size_t)tok * a.q_stride + (size_t)head * hd;
    half8 qh[KQ ? 1 : KS], ql[KQ ? 1 : KS];
    QuantQ<KQ ? KS : 1> qq;
    float c = a.scale * kLog2e;
    if constexpr (KQ)
        load_quant_q<KS>(a, q_row, live, g, qq);
    else
        c *= load_q<KS>(a, q_row, live, g, qh, ql);
    int vlo, vhi;
    row_sees(a, sc, pc, mi, vlo, vhi);
    const int full_lo = wave_max(vlo), full_hi = wave_min(vhi);
    const int krb = kv_row_bytes(a.k_fmt, hd), vrb = kv_row_bytes(a.v_fmt, hd);
    const int kblk = a.k_fmt == 1 ? 34 : 18, vblk = a.v_fmt == 1 ? 34 : 18;

    float m = -INFINITY, l = 0.0f;
    float4v o[NG][8];
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int d = 0; d < 8; ++d) o[n][d] = float4v{0, 0, 0, 0};

    auto place_of_lane = [&](int t0) {
        const int pos = t0 + (lane & 31);
        if (pos >= pc.p1) return -1;
        const int place = place_at(a, pc.table, pos);
        if (place < 0 && lane < 32) page_fault(a.faults);
        return place;
    };
    uint4 kf[KQ ? 1 : 2][KQ ? 1 : KS];
    Bytes8 kq[KQ ? 2 : 1][KQ ? KS : 1];
    uint16_t kd[KQ ? 2 : 1][KQ ? KS : 1];
    auto load_k = [&](int place) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint8_t *row = kv_row(a, a.k, krb, __shfl(place, 16 * h + i, 64), pc.kvh);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if constexpr (KQ) {
                    const uint8_t *b = row + (s * 32 < hd ? s * kblk : 0);
                    kd[h][s] = *reinterpret_cast<const uint16_t *>(b);
                    kq[h][s] = *reinterpret_cast<const Bytes8 *>(b + 2 + (a.k_fmt == 1 ? 8 * g : 8 * (g & 1)));
                } else {
                    kf[h][s] = *reinterpret_cast<const uint4 *>(row + g * 16 + (s * 32 < hd ? s * 64 : 0));
                }
            }
        }
    };
    int place = place_of_lane(pc.p0), place_next = place_of_lane(pc.p0 + kUnitA);
    load_k(place);
    for (int t0 = pc.p0; t0 < pc.p1; t0 += kUnitA) {
        const uint32_t there = (uint32_t)__ballot(place >= 0);  // bit p: position t0 + p
        lds.place[lane & 31] = place;
        const int4 pa = *reinterpret_cast<const int4 *>(lds.place + 4 * g);
        const int4 pb = *reinterpret_cast<const int4 *>(lds.place + 16 + 4 * g);
        const int pl[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
        uint4 v[VQ ? 1 : NG][8];
        Bytes8 vq[VQ ? NG : 1][8];
        _Float16 vd[VQ ? NG : 1][8];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const int d0 = n * 128 + 8 * i, dim = d0 < hd ? d0 : 0;  // past the head: the first dims, never stored
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint8_t *row = kv_row(a, a.v, vrb, pl[j], pc.kvh);
                if constexpr (VQ) {
                    const uint8_t *b = row + (dim >> 5) * vblk;
                    vd[n][j] = *reinterpret_cast<const _Float16 *>(b);
                    vq[n][j] = *reinterpret_cast<const Bytes8 *>(b + 2 + (a.v_fmt == 1 ? 8 * (i & 3) : 8 * (i & 1)));
                } else {
                    v[n][j] = *reinterpret_cast<const uint4 *>(row + dim * 2);
                }
            }
        }
        float x[8];
        if constexpr (KQ) {
            float4v acc[2] = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w0 = kq[h][s].a, w1 = kq[h][s].b;
                    if (a.k_fmt == 2) {  // dims 8 g .. of the block: low nibbles, then high ones
                        w0 = (w0 >> (4 * (g >> 1))) & 0x0f0f0f0fu;
                        w1 = (w1 >> (4 * (g >> 1))) & 0x0f0f0f0fu;
                    }
                    const long kk = (long)((uint64_t)w0 | ((uint64_t)w1 << 32));
                    const int4v is = __builtin_amdgcn_mfma_i32_16x16x32_i8(qq.q[s], kk, qq.sum8[s], 0, 0, 0);
                    const float dk = f16_bits_to_f32(kd[h][s]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[h][r] = fmaf((float)is[r], dk * qq.d[s][r], acc[h][r]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) lds.scores[(4 * g + r) * kTrRow + 16 * h + i] = acc[h][r];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 y = *reinterpret_cast<const float4 *>(lds.scores + i * kTrRow + 16 * h + 4 * g);
                x[4 * h] = y.x * c, x[4 * h + 1] = y.y * c, x[4 * h + 2] = y.z * c, x[4 * h + 3] = y.w * c;
            }
            __builtin_amdgcn_wave_barrier();
        } else {
            float4v acc[2][2] = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const half8 kk = __builtin_bit_cast(half8, kf[h][s]);
                    acc[h][0] = mfma(kk, qh[s], acc[h][0]);
                    acc[h][1] = mfma(kk, ql[s], acc[h][1]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[4 * h + r] = (acc[h][0][r] + acc[h][1][r]) * c;
        }
        const int place_2 = place_of_lane(t0 + 2 * kUnitA);
        if (t0 + kUnitA < pc.p1) load_k(place_next);
        const bool edge = t0 < full_lo || t0 + kUnitA > full_hi || there != 0xffffffffu;
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int p = 16 * (e >> 2) + 4 * g + (e & 3), pos = t0 + p;
                if (pos < vlo || pos >= vhi || !((there >> p) & 1)) x[e] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (pl[j] < 0) {  // nothing is there: whatever was read must not meet a weight of 0
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        if constexpr (VQ)
                            vd[n][j] = (_Float16)0.0f;
                        else
                            v[n][j] = make_uint4(0, 0, 0, 0);
                    }
                }
        }
        float f;
        if (softmax_step<8>(x, m, l, f)) {
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int d = 0; d < 8; ++d) o[n][d] *= f;
        }
        uint32_t ph[4], pw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split_p(x[2 * e], x[2 * e + 1], ph[e], pw[e]);
        const half8 p_hi = as_half8(ph[0], ph[1], ph[2], ph[3]), p_lo = as_half8(pw[0], pw[1], pw[2], pw[3]);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if constexpr (VQ) {
                // quants as unsigned bytes u, read as the f16 number 1024 + u, less 1024 and the bytes' offset
                const bool q8 = a.v_fmt == 1;
                const int sh = 4 * ((i & 3) >> 1);
                const half2v off = q8 ? half2v{(_Float16)-1152.0f, (_Float16)-1152.0f}
                                      : half2v{(_Float16)-1032.0f, (_Float16)-1032.0f};
                uint32_t w[8][2];
                half2v d2[4];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j][0] = q8 ? vq[n][j].a ^ 0x80808080u : (vq[n][j].a >> sh) & 0x0f0f0f0fu;
                    w[j][1] = q8 ? vq[n][j].b ^ 0x80808080u : (vq[n][j].b >> sh) & 0x0f0f0f0fu;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) d2[e] = half2v{vd[n][2 * e], vd[n][2 * e + 1]};
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
        place = place_next;
        place_next = place_2;
    }
    l = row_sum(l);
    float check = l;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int d = 0; d < 8; ++d) check += o[n][d][0] + o[n][d][1] + o[n][d][2] + o[n][d][3];
    check = row_sum(check);
    const bool wrong = live && check - check != 0.0f;  // NaN or infinite
    if (live && !wrong) {
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
        if (g == 0) to.ml[at] = make_float2(m - kShift, l);
    }
    uint32_t again = (uint32_t)__ballot(wrong) & 0xffffu;
    while (again) {
        const int b = __builtin_ctz(again);
        again &= again - 1;
        const size_t at = part_row(a, pc, to, pc.row0 + b);
        slow_row(a, pc, pc.row0 + b, __shfl(vlo, b, 64), __shfl(vhi, b, 64), to.o + at * hd, to.ml + at);
    }
}

// ---- block items: a workgroup, 128 query rows, K and V through LDS ------------------
//
// Tiles of T = 16384 / DP positions, two in LDS (128 KB): while the waves work on
// one, the next is under way.  K goes to LDS directly (global_load_lds), 16-byte
// pieces of a row exchanged by the position's low bits so that a wave's reads of
// 16 positions meet no bank twice; V is transposed on its way, as in a
// stream item, by the thread that has loaded 8 positions x 8 dims, and written as
// 16-byte runs of 8 positions, exchanged by the dim's low bits.  A wave holds 16 * R
// rows; each piece read from LDS feeds 2 * R products.

// K and V row runs of a block tile in LDS, in 16-byte pieces.
template <int T>
__device__ __forceinline__ int v_piece(int dim, int run)
{
    if constexpr (T >= 64)
        return dim * (T / 8) + (run ^ (dim & 7) ^ ((dim >> 3) & 7));
    else
        return dim * (T / 8) + (run ^ ((dim >> 1) & 3) ^ ((dim >> 3) & 3));
}

template <int DP>
struct BlockLds {
    static constexpr int T = 16384 / DP;
    uint4 k[2][2048], v[2][2048];
    int place[3][T];
};

template <int DP, int R>
__device__ __forceinline__ void block_item(const PagedAttn &a, const Scan &sc, const Piece &pc, BlockLds<DP> &lds,
                                           const Dest &to)
{
    constexpr int KS = DP / 32, NF = DP / 16, T = 16384 / DP, SP = T < 64 ? T : 64, NH = SP / 16, P = DP / 8;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4, hd = a.head_dim;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rb = hd * 2;
    const int tiles = (pc.p1 - pc.p0 + T - 1) / T;

    auto set_places = [&](int tile) {
        if (tid < T) {
            const int pos = pc.p0 + tile * T + tid;
            int place = -1;
            if (pos < pc.p1) {
                place = place_at(a, pc.table, pos);
                if (place < 0) page_fault(a.faults);
            }
            lds.place[tile % 3][tid] = place;
        }
    };
    auto load_k = [&](int tile) {
        // a wave's share: T / 4 positions, 64 pieces an instruction
        constexpr int PI = 64 / P > 0 ? 64 / P : 1;  // positions an instruction
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int p = wave * (T / 4) + n * PI + lane / P, piece = (lane % P) ^ (p & 7);
            const uint8_t *src = kv_row(a, a.k, rb, lds.place[tile % 3][p], pc.kvh) + (piece * 8 < hd ? piece * 16 : 0);
            uint4 *dst = &lds.k[tile & 1][(wave * (T / 4) + n * PI) * P];
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)src,
                                             (__attribute__((address_space(3))) uint32_t *)dst, 16, 0, 0);
        }
    };
    const int dl = tid % P, run = tid / P;  // this thread's dims 8 dl .. and run of positions
    constexpr int kTasks = (T / 8) * P;     // 256
    static_assert(kTasks == 256, "one task a thread");
    const int run0 = (run >> 2) * 32 + (run & 3) * 4;  // positions run0 + 0..3 and run0 + 16..19
    uint4 v[8];
    int vp[8];
    auto load_v = [&](int tile) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            vp[j] = lds.place[tile % 3][run0 + (j >> 2) * 16 + (j & 3)];
            v[j] = *reinterpret_cast<const uint4 *>(kv_row(a, a.v, rb, vp[j], pc.kvh) + (dl * 8 < hd ? dl * 16 : 0));
        }
    };
    auto store_v = [&](int tile) {
        uint32_t w[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t keep = vp[j] < 0 ? 0u : 0xffffffffu;  // nothing there: no weight may meet it
            w[j][0] = v[j].x & keep, w[j][1] = v[j].y & keep, w[j][2] = v[j].z & keep, w[j][3] = v[j].w & keep;
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
            uint32_t t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = __builtin_amdgcn_perm(w[2 * e + 1][d >> 1], w[2 * e][d >> 1], sel);
            lds.v[tile & 1][v_piece<T>(8 * dl + d, run)] = make_uint4(t[0], t[1], t[2], t[3]);
        }
    };

    __syncthreads();  // the tiles' LDS is free
    set_places(0);
    if (tiles > 1) set_places(1);
    __syncthreads();
    if (tiles > 0) {
        load_k(0);
        load_v(0);
    }

    half8 qh[R][KS], ql[R][KS];
    float c[R], m[R], l[R];
    int vlo[R], vhi[R], full_lo = 0, full_hi = INT32_MAX;
    float4v o[R][NF];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int mi = pc.row0 + (wave * R + u) * 16 + i;
        const bool live = mi < pc.rows;
        const int tok = pc.tok0 + mi / a.group, head = pc.kvh * a.group + mi % a.group;
        c[u] = load_q<KS>(a, a.q + (size_t)tok * a.q_stride + (size_t)head * hd, live, g, qh[u], ql[u]) * a.scale * kLog2e;
        row_sees(a, sc, pc, mi, vlo[u], vhi[u]);
        full_lo = max(full_lo, wave_max(vlo[u]));
        full_hi = min(full_hi, wave_min(vhi[u]));
        m[u] = -INFINITY;
        l[u] = 0.0f;
#pragma unroll
        for (int f = 0; f < NF; ++f) o[u][f] = float4v{0, 0, 0, 0};
    }
    if (tiles > 0) store_v(0);

    for (int tile = 0; tile < tiles; ++tile) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): K of this tile is in LDS
        __syncthreads();
        if (tile + 2 < tiles) set_places(tile + 2);
        if (tile + 1 < tiles) {
            load_k(tile + 1);
            load_v(tile + 1);
        }
        const uint4 *kt = lds.k[tile & 1], *vt = lds.v[tile & 1];
#pragma unroll 1
        for (int s0 = 0; s0 < T; s0 += SP) {
            const int t0 = pc.p0 + tile * T + s0;
            if (t0 >= pc.p1) break;
            float4v acc[R][NH];
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int h = 0; h < NH; ++h) acc[u][h] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const int p = s0 + 16 * h + i;
                    const half8 kk = __builtin_bit_cast(half8, kt[p * P + ((4 * s + g) ^ (p & 7))]);
#pragma unroll
                    for (int u = 0; u < R; ++u) acc[u][h] = mfma(kk, qh[u][s], acc[u][h]);
#pragma unroll
                    for (int u = 0; u < R; ++u) acc[u][h] = mfma(kk, ql[u][s], acc[u][h]);
                }
            }
            const uint64_t there = __ballot(lane < SP && lds.place[tile % 3][s0 + (lane & (SP - 1))] >= 0);
            const bool edge = t0 < full_lo || t0 + SP > full_hi || there != (SP == 64 ? ~0ull : (1ull << (SP & 63)) - 1);
            uint32_t ph[R][NH][2], pw[R][NH][2];
#pragma unroll
            for (int u = 0; u < R; ++u) {
                float x[4 * NH];
#pragma unroll
                for (int e = 0; e < 4 * NH; ++e) x[e] = acc[u][e >> 2][e & 3] * c[u];
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 4 * NH; ++e) {
                        const int p = 16 * (e >> 2) + 4 * g + (e & 3), pos = t0 + p;
                        if (pos < vlo[u] || pos >= vhi[u] || !((there >> p) & 1)) x[e] = -INFINITY;
                    }
                }
                float f;
                if (softmax_step<4 * NH>(x, m[u], l[u], f)) {
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
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const half8 vv = __builtin_bit_cast(half8, vt[v_piece<T>(16 * f + i, s0 / 8 + 4 * b + g)]);
#pragma unroll
                    for (int u = 0; u < R; ++u) o[u][f] = mfma(vv, p_hi[u], o[u][f]);
#pragma unroll
                    for (int u = 0; u < R; ++u) o[u][f] = mfma(vv, p_lo[u], o[u][f]);
                }
            }
        }
        if (tile + 1 < tiles) store_v(tile + 1);
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int first = pc.row0 + (wave * R + u) * 16, mi = first + i;
        const bool live = mi < pc.rows;
        const float lu = row_sum(l[u]);
        float check = lu;
#pragma unroll
        for (int f = 0; f < NF; ++f) check += o[u][f][0] + o[u][f][1] + o[u][f][2] + o[u][f][3];
        check = row_sum(check);
        const bool wrong = live && check - check != 0.0f;  // NaN or infinite
        if (live && !wrong) {
            const size_t at = part_row(a, pc, to, mi);
            float *dst = to.o + at * hd;
#pragma unroll
            for (int f = 0; f < NF; ++f)
                if (f * 16 < hd)
                    *reinterpret_cast<float4 *>(dst + 16 * f + 4 * g) =
                        make_float4(o[u][f][0], o[u][f][1], o[u][f][2], o[u][f][3]);
            if (g == 0) to.ml[at] = make_float2(m[u] - kShift, lu);
        }
        uint32_t again = (uint32_t)__ballot(wrong) & 0xffffu;
        while (again) {
            const int b = __builtin_ctz(again);
            again &= again - 1;
            const size_t at = part_row(a, pc, to, first + b);
            slow_row(a, pc, first + b, __shfl(vlo[u], b, 64), __shfl(vhi[u], b, 64), to.o + at * hd, to.ml + at);
        }
    }
}

// ---- the launch --------------------------------------------------------------------

// The prefix's items: of the batch's rows, in one kind.
struct Shared {
    int rows;              // rows x group
    bool few;              // stream items
    int lo, hi;            // positions any row sees
    int units, blocks;     // units an item, row blocks
};

__device__ __forceinline__ Shared shared_work(const PagedAttn &a, const Scan &s, bool blocks, int unit)
{
    Shared p;
    p.rows = (s.rs[kScanT] - s.rs[0]) * a.group;
    p.few = !blocks || p.rows <= kFewRows;
    p.hi = a.prefix_len;
    p.lo = 0;
    if (a.window && s.low < INT32_MAX) p.lo = min(max(a.prefix_len + s.low - a.window + 1, 0), p.hi);
    const int tile = p.few ? kRowsA : kRowsB;
    p.blocks = a.prefix_len > 0 ? (p.rows + tile - 1) / tile : 0;
    p.units = units_of(p.lo, p.hi, p.few ? kUnitA : unit);
    return p;
}

// The piece at unit u of the stream or block items, at most `left` units long;
// returns the units taken, and the item's index, and whether the piece holds
// its first and last unit.
__device__ __forceinline__ int find_piece(const PagedAttn &a, const Scan &s, const Shared &sh, bool blocks, bool block,
                                          int unit, int u, int left, Piece &pc, int &item, bool &is_first, bool &is_last)
{
    const int tile = block ? kRowsB : kRowsA, step = block ? unit : kUnitA;
    const bool sh_here = sh.few != block;
    const int sh_items = sh_here ? sh.blocks * a.n_kv_heads : 0;
    const int sh_units = sh_items * sh.units;
    int lo, hi, units, within, blk;
    if (u < sh_units) {
        item = u / sh.units;
        within = u - item * sh.units;
        blk = item / a.n_kv_heads;
        units = sh.units;
        lo = sh.lo;
        hi = sh.hi;
        pc.pre = true;
        pc.table = a.prefix;
        pc.tok0 = s.rs[0];
        pc.rows = sh.rows;
        pc.at0 = 0;
    } else {
        u -= sh_units;
        const int per = (a.n_seqs + kScanT - 1) / kScanT;
        const int t = share_of(block ? s.ub : s.ua, u);
        int r = t * per, at = (block ? s.ub : s.ua)[t], first = (block ? s.ib : s.ia)[t];
        Request q;
        int w[4];
        for (;; ++r) {
            q = request_at(a, r);
            request_work(a, q, blocks, unit, w);
            const int n = block ? w[1] : w[0];
            if (u < at + n || r + 1 >= a.n_seqs) break;
            at += n;
            first += block ? w[3] : w[2];
        }
        u -= at;
        if (!block) {
            units = own_units_a(a, q);
            item = u / units;
            within = u - item * units;
            blk = item / a.n_kv_heads;
            own_range(a, q, 0, q.n - 1, lo, hi);
        } else {
            blk = 0;
            for (;; ++blk) {
                units = own_units_b(a, q, blk, unit);
                if (u < units * a.n_kv_heads) break;
                u -= units * a.n_kv_heads;
            }
            const int kv = u / units;
            item = blk * a.n_kv_heads + kv;
            within = u - kv * units;
            const int last = min(q.n * a.group, (blk + 1) * kRowsB) - 1;
            own_range(a, q, blk * kRowsB / a.group, last / a.group, lo, hi);
        }
        pc.pre = false;
        pc.table = a.table + (size_t)r * a.table_stride;
        pc.tok0 = q.rs;
        pc.rows = q.n * a.group;
        pc.at0 = q.len - q.n;
        const int kvh_item = item;
        item += sh_items + first;
        pc.kvh = kvh_item % a.n_kv_heads;
        blk = kvh_item / a.n_kv_heads;
    }
    if (pc.pre) pc.kvh = item % a.n_kv_heads;
    pc.row0 = blk * tile;
    const int take = min(units - within, left);
    pc.p0 = lo + within * step;
    pc.p1 = min(hi, pc.p0 + take * step);
    is_first = within == 0;
    is_last = within + take == units;
    return take;
}

template <int DP, bool KQ, bool VQ, int R>
struct KernelLds {
    Scan scan;
    union {
        WaveLds wave[4];
        BlockLds<DP> block;
    };
};
template <int DP, bool KQ, bool VQ>
struct KernelLds<DP, KQ, VQ, 0> {
    Scan scan;
    WaveLds wave[4];
};

// R: rows of a block item's wave / 16 (0: stream items alone, the quantised caches).
template <int DP, bool KQ, bool VQ, int R>
__global__ __launch_bounds__(kScanT, 1) void paged_attn_kernel(PagedAttn a, Parts parts)
{
    __shared__ KernelLds<DP, KQ, VQ, R> lds;
    constexpr bool kBlocks = R > 0;
    constexpr int kUnitB = unit_b(DP);
    const Scan &s = lds.scan;
    scan_requests(a, lds.scan, kBlocks, kUnitB);
    const int wg = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Shared sh{};
    // row starts that do not ascend, or more units than an int counts (days of work): nothing is computed
    bool bad = s.bad;
    if (!bad) {
        sh = shared_work(a, s, kBlocks, kUnitB);
        bad = s.size + (float)sh.blocks * (float)a.n_kv_heads * (float)sh.units > 1e9f;
    }
    if (wg == 0 && tid == 0) {
        parts.head[0] = !bad;
        parts.head[1] = bad ? 0 : s.rs[0];
        parts.head[2] = bad ? 0 : s.rs[kScanT];
        if (bad) page_fault(a.faults);
    }
    if (bad) return;
    const int sh_units = sh.blocks * a.n_kv_heads * sh.units, sh_items = sh.blocks * a.n_kv_heads;
    const int ua = s.ua[kScanT] + (sh.few ? sh_units : 0), ub = s.ub[kScanT] + (sh.few ? 0 : sh_units);

    // which items a row's own part is in
    for (int row = s.rs[0] + wg * kScanT + tid; row < s.rs[kScanT]; row += parts.wgs * kScanT) {
        const int r = request_of(a, s, row), per = (a.n_seqs + kScanT - 1) / kScanT, t = r / per;
        int ia = s.ia[t], ib = s.ib[t], w[4];
        for (int x = t * per; x < r; ++x) {
            request_work(a, request_at(a, x), kBlocks, kUnitB, w);
            ia += w[2];
            ib += w[3];
        }
        const Request q = request_at(a, r);
        const bool block = kBlocks && q.n * a.group > kFewRows;
        const int first = block ? parts.items_a + ib + (sh.few ? 0 : sh_items) : ia + (sh.few ? sh_items : 0);
        parts.row_item[row] = make_int2(first, (row - q.rs) | (block ? 1 << 30 : 0));
    }

    int wb = 0;
    if (ub > 0) {
        wb = parts.wgs;
        if (ua > 0) {
            const float fb = (float)ub * kCostB, fa = (float)ua * kCostA * 0.25f;
            wb = min(max((int)(parts.wgs * fb / (fa + fb) + 0.5f), 1), parts.wgs - 1);
        }
    }
    const int n_a = (parts.wgs - wb) * 4;
    Piece pc;
    int item;
    bool first, last;
    if constexpr (kBlocks) {
        if (wg < wb) {
            const int quota = (ub + wb - 1) / wb, end = min(ub, (wg + 1) * quota);
            for (int u = wg * quota; u < end;) {
                u += find_piece(a, s, sh, kBlocks, true, kUnitB, u, end - u, pc, item, first, last);
                const size_t row = (size_t)wg * kRowsB;
                const Dest to = first ? Dest{parts.o[!pc.pre], parts.ml[!pc.pre], true}
                                      : Dest{parts.o_b + row * a.head_dim, parts.ml_b + row, false};
                if (tid == 0 && first) parts.first[parts.items_a + item] = wg;
                if (tid == 0 && last) parts.last[parts.items_a + item] = wg;
                block_item<DP, R ? R : 1>(a, s, pc, lds.block, to);
            }
            return;
        }
    }
    const int worker = (wg - wb) + (parts.wgs - wb) * wave;
    const int quota = (ua + n_a - 1) / n_a, end = min(ua, (worker + 1) * quota);
    for (int u = worker * quota; u < end;) {
        u += find_piece(a, s, sh, kBlocks, false, kUnitB, u, end - u, pc, item, first, last);
        const size_t row = (size_t)worker * kRowsA;
        const Dest to = first ? Dest{parts.o[!pc.pre], parts.ml[!pc.pre], true}
                              : Dest{parts.o_a + row * a.head_dim, parts.ml_a + row, false};
        if ((tid & 63) == 0 && first) parts.first[item] = worker;
        if ((tid & 63) == 0 && last) parts.last[item] = worker;
        stream_item<DP, KQ, VQ>(a, s, pc, lds.wave[wave], to);
    }
}

// Joins the parts of each row and head: a workgroup a row and head, waves over
// the parts, lanes over the dims.
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn a, Parts parts, bool blocks)
{
    __shared__ float s_o[4][512], s_m[4], s_l[4];
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hd = a.head_dim;
    const int row0 = parts.head[1], row1 = parts.head[2];
    if (!parts.head[0] || row < row0 || row >= row1) return;
    const int kvh = h / a.group, gq = h - kvh * a.group;
    const size_t base = (size_t)row * a.n_heads + h;
    // the two items of the row: the prefix's, its own
    int w0[2], n[2], at[2];
    bool blk[2];
    {
        const int m = (row1 - row0) * a.group, mi = (row - row0) * a.group + gq;
        blk[0] = blocks && m > kFewRows;
        const int tile = blk[0] ? kRowsB : kRowsA, item = mi / tile * a.n_kv_heads + kvh + (blk[0] ? parts.items_a : 0);
        at[0] = mi % tile;
        w0[0] = a.prefix_len > 0 ? parts.first[item] : 0;
        n[0] = a.prefix_len > 0 ? parts.last[item] - w0[0] + 1 : 0;
    }
    {
        const int2 ri = parts.row_item[row];
        blk[1] = ri.y >> 30;
        const int mi = (ri.y & ~(1 << 30)) * a.group + gq, tile = blk[1] ? kRowsB : kRowsA;
        const int item = ri.x + mi / tile * a.n_kv_heads + kvh;
        at[1] = mi % tile;
        w0[1] = parts.first[item];
        n[1] = parts.last[item] - w0[1] + 1;
    }
    float m = -INFINITY, l = 0.0f;
    float o[8] = {};
    for (int k = wave; k < n[0] + n[1]; k += 4) {
        const int x = k >= n[0], j = k - (x ? n[0] : 0);
        const float *po;
        float2 ml;
        if (j == 0) {
            po = parts.o[x] + base * hd;
            ml = parts.ml[x][base];
        } else {
            const size_t r = (size_t)(w0[x] + j) * (blk[x] ? kRowsB : kRowsA) + at[x];
            po = (blk[x] ? parts.o_b : parts.o_a) + r * hd;
            ml = (blk[x] ? parts.ml_b : parts.ml_a)[r];
        }
        if (ml.y == 0.0f) continue;  // saw nothing
        const float m2 = fmaxf(m, ml.x), f = m == -INFINITY ? 0.0f : exp2f(m - m2), w = exp2f(ml.x - m2);
        l = l * f + ml.y * w;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e * 64 + lane < hd) o[e] = o[e] * f + po[e * 64 + lane] * w;
        m = m2;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e * 64 + lane < hd) s_o[wave][e * 64 + lane] = o[e];
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float f[4], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = s_l[w] == 0.0f ? 0.0f : exp2f(s_m[w] - top);
        sum += s_l[w] == 0.0f ? 0.0f : s_l[w] * f[w];
    }
    for (int d = tid; d < hd; d += 256) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) x += f[w] == 0.0f ? 0.0f : s_o[w][d] * f[w];
        a.out[base * hd + d] = sum == 0.0f ? 0.0f : x / sum;
    }
}

bool has_blocks(const PagedAttn &a) { return a.k_fmt == 0 && a.v_fmt == 0; }

Parts layout(const PagedAttn &a, uint8_t *base, size_t &bytes)
{
    Parts p{};
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t *x = base + at;
        at += align_up(n, 256);
        return x;
    };
    p.wgs = 256;
    const size_t heads = (size_t)a.max_rows * a.n_heads, hd = a.head_dim;
    const size_t group_rows = (size_t)a.max_rows * a.group;
    // stream items: the rows of every request and of the prefix in tiles of 16; block items: tiles of 128 of
    // groups of more than kFewRows
    const size_t seqs = std::min<size_t>(a.n_seqs, a.max_rows);
    const size_t items_a = (group_rows / kRowsA + seqs + group_rows / kRowsA + 1) * a.n_kv_heads;
    const size_t items_b = has_blocks(a) ? (2 * (group_rows / kRowsB + 1) + std::min(seqs, group_rows / kFewRows)) * a.n_kv_heads : 0;
    p.items_a = (int)items_a;
    for (int k = 0; k < 2; ++k) {
        const bool used = k == 1 || a.prefix_len > 0;
        p.o[k] = reinterpret_cast<float *>(take(used ? heads * hd * 4 : 0));
        p.ml[k] = reinterpret_cast<float2 *>(take(used ? heads * 8 : 0));
    }
    p.o_a = reinterpret_cast<float *>(take((size_t)p.wgs * 4 * kRowsA * hd * 4));
    p.ml_a = reinterpret_cast<float2 *>(take((size_t)p.wgs * 4 * kRowsA * 8));
    const size_t rows_b = has_blocks(a) ? (size_t)p.wgs * kRowsB : 0;
    p.o_b = reinterpret_cast<float *>(take(rows_b * hd * 4));
    p.ml_b = reinterpret_cast<float2 *>(take(rows_b * 8));
    p.first = reinterpret_cast<int32_t *>(take((items_a + items_b) * 4));
    p.last = reinterpret_cast<int32_t *>(take((items_a + items_b) * 4));
    p.row_item = reinterpret_cast<int2 *>(take((size_t)a.max_rows * 8));
    p.head = reinterpret_cast<int32_t *>(take(16));
    bytes = at;
    return p;
}

template <int DP, int R>
void launch_dp(mrml_hip_ctx *ctx, const PagedAttn &a, const Parts &p)
{
    const dim3 grid(p.wgs), block(kScanT);
    const bool kq = a.k_fmt != 0, vq = a.v_fmt != 0;
    if (!kq && !vq)
        hipLaunchKernelGGL((paged_attn_kernel<DP, false, false, R>), grid, block, 0, ctx->stream, a, p);
    else if (!kq)
        hipLaunchKernelGGL((paged_attn_kernel<DP, false, true, 0>), grid, block, 0, ctx->stream, a, p);
    else if (!vq)
        hipLaunchKernelGGL((paged_attn_kernel<DP, true, false, 0>), grid, block, 0, ctx->stream, a, p);
    else
        hipLaunchKernelGGL((paged_attn_kernel<DP, true, true, 0>), grid, block, 0, ctx->stream, a, p);
}

}  // namespace

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
    if (a.head_dim <= 64)
        launch_dp<64, 2>(ctx, a, p);
    else if (a.head_dim <= 128)
        launch_dp<128, 2>(ctx, a, p);
    else if (a.head_dim <= 256)
        launch_dp<256, 2>(ctx, a, p);
    else
        launch_dp<512, 1>(ctx, a, p);
    if (int rc = check_launch(ctx, "paged_attn_kernel")) return rc;
    hipLaunchKernelGGL(paged_merge_kernel, dim3(a.max_rows, a.n_heads), dim3(256), 0, ctx->stream, a, p, has_blocks(a));
    return check_launch(ctx, "paged_merge_kernel");
}

}  // namespace mrml
