// moe.hip -- a mixture-of-experts layer for a batch of tokens, around the
// experts' products (moe_ffn.hip): the residual's addition and norm, the
// router's logits, the route, and the C ABI of them all.

#include <algorithm>
#include <cmath>

#include "moe.h"
#include "norm_block.h"

namespace mrml {

namespace {

using f32x4 = float __attribute__((ext_vector_type(4)));

constexpr int kOneRoute = 16;  // tokens that one workgroup routes and plans

// ---- residual and norm -----------------------------------------------------------

// v of the lane that a DPP control names, as two words; 0 where it names none or ROWS leaves the row out.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ double lane_f64(double v, int lane)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over the wave, in a fixed order: within rows of 16 lanes, then rows 0 and 1, 2 and 3, then both halves.
__device__ __forceinline__ double wave_sum_f64(double v)
{
    v += dpp_f64<0xB1>(v);        // quad_perm 1,0,3,2
    v += dpp_f64<0x4E>(v);        // quad_perm 2,3,0,1
    v += dpp_f64<0x124>(v);       // row_ror:4
    v += dpp_f64<0x128>(v);       // row_ror:8
    v += dpp_f64<0x142, 0xa>(v);  // row_bcast:15
    v += dpp_f64<0x143, 0xc>(v);  // row_bcast:31
    return lane_f64(v, 63);
}

// Sum over the workgroup; red: a double a wave, free again after the next barrier.
__device__ __forceinline__ double block_sum_f64(double v, double *red)
{
    v = wave_sum_f64(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += red[w];
    return s;
}

__device__ __forceinline__ double sq_f64(float4 a)
{
    return ((double)a.x * a.x + (double)a.y * a.y) + ((double)a.z * a.z + (double)a.w * a.w);
}

// One workgroup a row, CH float4 a thread: each value is read once, and waits in registers for the sums of its row.  The sums
// are f64, so that their order leaves no trace in the f32 scale, nor in the quants behind it.  1900 rows of 2304 with a pack:
// 15.9 us, 4.7 TB/s, bound by its bytes; one row: 4.8, a launch and the latencies of a load and two sums.
template <int CH, int THREADS>
__global__ __launch_bounds__(THREADS) void residual_norm_rows_kernel(const float *t, const float *__restrict__ w_post,
                                                                 const float *h, float *h_out,
                                                                 const float *__restrict__ w_next, float *xn,
                                                                 uint8_t *__restrict__ pack, int dim, float eps,
                                                                 int norm_t)
{
    __shared__ double red[2][THREADS / 64];
    const int n4 = dim >> 2, nb = dim >> 5;
    const size_t row = blockIdx.x, at = row * n4;
    const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float4 v[CH], hv[CH], wp[CH], wn[CH];
    load_w<CH>(norm_t ? w_post : nullptr, wp, n4);
    load_w<CH>(w_next, wn, n4);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const int c = threadIdx.x + k * blockDim.x;
        v[k] = c < n4 ? reinterpret_cast<const float4 *>(t)[at + c] : zero;
        hv[k] = c < n4 ? reinterpret_cast<const float4 *>(h)[at + c] : zero;
        s += sq_f64(v[k]);
    }
    if (norm_t) {
        const float scale = rms_scale((float)(block_sum_f64(s, red[0]) / (double)dim), 1, eps);
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            v[k] = scale4(v[k], scale);
            if (w_post) v[k] = mul4(v[k], wp[k]);
        }
    }
    s = 0.0;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const int c = threadIdx.x + k * blockDim.x;
        v[k] = add4(hv[k], v[k]);
        if (c < n4) reinterpret_cast<float4 *>(h_out)[at + c] = v[k];
        s += c < n4 ? sq_f64(v[k]) : 0.0;
    }
    if (!xn && !pack) return;
    const float scale = rms_scale((float)(block_sum_f64(s, red[1]) / (double)dim), 1, eps);
    const size_t all = (size_t)gridDim.x * nb;  // blocks of the whole pack
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const int c = threadIdx.x + k * blockDim.x;
        float4 o = scale4(v[k], scale);
        if (w_next) o = mul4(o, wn[k]);
        if (xn && c < n4) reinterpret_cast<float4 *>(xn)[at + c] = o;
        if (pack) {
            uint32_t dbits;
            int sum;
            const uint32_t q = q8_0_block8x4(o, dbits, sum);
            const size_t b = row * nb + (c >> 3);
            if (c < n4) {
                reinterpret_cast<uint32_t *>(pack)[at + c] = q;
                if ((c & 7) == 0) {
                    reinterpret_cast<float *>(pack + all * 32)[b] = f16_bits_to_f32(dbits);
                    reinterpret_cast<int32_t *>(pack + all * 36)[b] = sum;
                }
            }
        }
    }
}

// ---- the router's product ----------------------------------------------------------

// For a few tokens: one wave a token and expert.
__global__ __launch_bounds__(256) void moe_logits_kernel(const float *__restrict__ x, const float *__restrict__ w,
                                                         float *__restrict__ logits, int n_experts, int cols, int batch)
{
    const int e = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (e >= n_experts) return;
    const float4 *a = reinterpret_cast<const float4 *>(x + (size_t)blockIdx.x * cols);
    const float4 *b = reinterpret_cast<const float4 *>(w + (size_t)e * cols);
    float s = 0.0f;
    for (int c = lane; c < cols / 4; c += 64) {
        const float4 u = a[c], v = b[c];
        s += (u.x * v.x + u.y * v.y) + (u.z * v.z + u.w * v.w);
    }
    s = mrml_xsum::wave_sum_f32(s);
    if (lane == 0) logits[(size_t)blockIdx.x * n_experts + e] = s;
}

// For more: a workgroup makes T * 16 tokens by T * 16 experts on f32 MFMA, its eight waves every eighth block of 32
// columns each, and adds the eight partial products.  The lanes of an operand's row are 16 or 32 apart, so that next lanes
// hold other rows, and a load of that form fetches 16 bytes a clock (51 us for the case below).  Whole lines of 8 rows an
// instruction therefore go through LDS, each wave through a part of its own (no barrier), 16-byte column c of row r at
// c ^ r % 8 so that the rows of a read lie in different banks.  A lane reads 16 bytes: component j of a row's lanes are
// the columns that MFMA j takes, of x and w alike.
// 1999 tokens, 128 experts of 2816 columns: 17.9 us (one wave a token and expert: 173), against 9.2 that f32 MFMA takes
// for them and 4.7 for the bytes; the loads' way through L1 and LDS, about as long again, hides behind the MFMA only in part.
// T = 2 reads half as much a product; T = 1 fills the chip with fewer tokens.  128 experts, T = 1 / 2: 64 tokens 6.7 / 16.9
// us, 512 6.9 / 17.5, 1024 11.7 / 17.5, 1999 20.9 / 17.9; 512 experts: 256 13.7 / 17.8, 512 26.3 / 18.1, 1999 94.4 / 65.0.
template <int T>
__global__ __launch_bounds__(512) void moe_logits_tile_kernel(const float *__restrict__ x, const float *__restrict__ w,
                                                              float *__restrict__ logits, int n_experts, int cols,
                                                              int batch)
{
    constexpr int S = T * 16, K = 64 / S, W = 8;  // rows, lanes a row, waves
    using Acc = float __attribute__((ext_vector_type(S * S / 64)));
    union Shared {
        f32x4 lines[W][2 * S * 8];
        float part[W][S][S + 1];
    };
    __shared__ Shared sh;
    // the tiles of one group of tokens on one XCD (workgroups go to the eight in turn), whose L2 then reads them once
    const int across = (n_experts + S - 1) / S, id = blockIdx.x / 8;
    const int t0 = (id / across * 8 + blockIdx.x % 8) * S, e0 = id % across * S;
    if (t0 >= batch) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int m = lane % S, g = lane / S, row = lane >> 3, chunks = cols / 32, n = (chunks - wave + W - 1) / W;
    const float *p[4 * T];
#pragma unroll
    for (int i = 0; i < 2 * T; ++i) {  // rows behind the last one read that one; their results are not stored
        p[i] = x + (size_t)min(t0 + i * 8 + row, batch - 1) * cols + (lane & 7) * 4;
        p[2 * T + i] = w + (size_t)min(e0 + i * 8 + row, n_experts - 1) * cols + (lane & 7) * 4;
    }
    f32x4 *mine = sh.lines[wave];
    f32x4 next[2][4 * T];
    auto load = [&](f32x4 (&v)[4 * T], int i) {
        const int at = min(wave + i * W, chunks - 1) * 32;
#pragma unroll
        for (int r = 0; r < 4 * T; ++r) v[r] = *reinterpret_cast<const f32x4 *>(p[r] + at);
        __builtin_amdgcn_sched_barrier(0);  // loads stay in this order, so that a wait leaves the later ones out
    };
    Acc acc[2] = {};
    auto product = [&](const f32x4 (&v)[4 * T]) {
#pragma unroll
        for (int r = 0; r < 4 * T; ++r) mine[r * 64 + row * 8 + ((lane ^ row) & 7)] = v[r];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 2 * T; ++i) {
            const f32x4 a = mine[m * 8 + ((i * K + g) ^ (m & 7))], b = mine[(S + m) * 8 + ((i * K + g) ^ (m & 7))];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (T == 2) acc[j & 1] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc[j & 1], 0, 0, 0);
                else acc[j & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc[j & 1], 0, 0, 0);
            }
        }
        __builtin_amdgcn_wave_barrier();
    };
    load(next[0], 0);
    for (int i = 0; i + 1 < n; i += 2) {
        load(next[1], i + 1);
        product(next[0]);
        load(next[0], i + 2);
        product(next[1]);
    }
    if (n & 1) product(next[0]);
    acc[0] += acc[1];
    __syncthreads();  // the parts lie where the lines did
#pragma unroll
    for (int r = 0; r < T * T * 4; ++r) sh.part[wave][r / 4 * 8 + g * 4 + r % 4][m] = acc[0][r];
    __syncthreads();
    for (int i = threadIdx.x; i < S * S; i += W * 64) {
        const int t = i / S, e = i % S;
        float s = sh.part[0][t][e];
#pragma unroll
        for (int v = 1; v < W; ++v) s += sh.part[v][t][e];
        if (t0 + t < batch && e0 + e < n_experts) logits[(size_t)(t0 + t) * n_experts + e0 + e] = s;
    }
}

// ---- the route -----------------------------------------------------------------------

// A value as a number whose order is the values': 0 for one that cannot be chosen (switched off, not a number, the
// lowest infinity), which no other value gives.  Both zeros give the same.
__device__ __forceinline__ uint64_t sort_key(double v)
{
    if (!(v > -INFINITY)) return 0;
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

__device__ __forceinline__ double key_value(uint64_t k)
{
    return k == 0 ? -INFINITY : __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
    auto step = [](uint32_t a, int b) { return max(a, (uint32_t)b); };
    v = step(v, dpp_mov<0xB1>((int)v));
    v = step(v, dpp_mov<0x4E>((int)v));
    v = step(v, dpp_mov<0x124>((int)v));
    v = step(v, dpp_mov<0x128>((int)v));
    v = step(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
    v = step(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane((int)v, 63);
}

// The lane that holds the largest key, of equal ones that with the lowest id; -1 if every key is 0.  Two keys seldom
// agree in their upper halves, so one maximum over 32 bits mostly decides.
__device__ __forceinline__ int wave_first(uint64_t key, int id)
{
    const uint32_t hi = wave_max_u32(key >> 32);
    if (hi == 0) return -1;
    uint64_t lanes = __ballot((uint32_t)(key >> 32) == hi);
    if (lanes & (lanes - 1)) {
        bool in = (uint32_t)(key >> 32) == hi;
        const uint32_t lo = wave_max_u32(in ? (uint32_t)key : 0);
        in = in && (uint32_t)key == lo;
        const uint32_t first = wave_max_u32(in ? ~(uint32_t)id : 0);
        lanes = __ballot(in && ~(uint32_t)id == first);
    }
    return __ffsll((unsigned long long)lanes) - 1;
}

// (32008 ids of 256 experts, 32 workgroups: 8.4 to 8.8 us, most of it the counting, an addition in LDS for every id in every
// workgroup; one workgroup an expert that looks through all ids twice took 73.)
// The plan of places [lo, hi) of n ids, by a workgroup of whole waves, at most 16: counts of every expert, before lo and
// in all, give where its run goes on; then, blockDim.x ids at a time, a place is its run's end, the ids of the same
// expert in lower waves and those in lower lanes.  Additions to the counters are whole numbers, so their order does not
// matter.  The workgroup with lo = 0 writes the starts as well.
struct PlanShared {
    int count[2][kMaxExperts];          // of ids before lo, and from lo on; then count[0]: where the run goes on
    int waves[16 * kMaxExperts];        // of a wave's ids of one expert in the present part
    int sums[16];
};

__device__ __forceinline__ void plan_range(const int32_t *ids, int32_t *__restrict__ starts, int32_t *__restrict__ order,
                                           int n_experts, int n, int lo, int hi, PlanShared &sh)
{
    constexpr int kAhead = 8;  // loads in flight
    const int threads = blockDim.x, wave = threadIdx.x >> 6, n_waves = threads >> 6, lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e < n_experts; e += threads) sh.count[0][e] = sh.count[1][e] = 0;
    for (int i = threadIdx.x; i < n_waves * n_experts; i += threads) sh.waves[i] = 0;
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < n; i0 += threads * kAhead) {
        int id[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) id[u] = i0 + u * threads < n ? ids[i0 + u * threads] : -1;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (id[u] >= 0) atomicAdd(&sh.count[i0 + u * threads >= lo][id[u]], 1);
    }
    __syncthreads();
    int base = 0;  // the runs of a thread's experts, threads at a time
    for (int e0 = 0; e0 < n_experts; e0 += threads) {
        const int e = e0 + threadIdx.x, before = e < n_experts ? sh.count[0][e] : 0;
        const int all = e < n_experts ? before + sh.count[1][e] : 0;
        int upto = all;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int v = __shfl_up(upto, d, 64);
            if (lane >= d) upto += v;
        }
        if (lane == 63) sh.sums[wave] = upto;
        __syncthreads();
        int start = base + upto - all;
        for (int w = 0; w < n_waves; ++w) {
            if (w < wave) start += sh.sums[w];
            base += sh.sums[w];
        }
        if (e < n_experts) {
            sh.count[0][e] = start + before;
            if (lo == 0) starts[e] = start;
        }
        __syncthreads();
    }
    if (lo == 0 && threadIdx.x == 0) starts[n_experts] = base;
    for (int i = max(lo, base) + threadIdx.x; i < hi; i += threads) order[i] = -1;
    for (int i0 = lo; i0 < hi; i0 += threads) {
        const int i = i0 + threadIdx.x, id = i < hi ? ids[i] : -1;
        uint64_t same = __ballot(id >= 0);
        for (int b = 0; (1 << b) < n_experts; ++b) {
            const bool set = (id >> b) & 1;
            const uint64_t with = __ballot(set);
            same &= set ? with : ~with;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (id >= 0 && rank == 0) sh.waves[wave * n_experts + id] = __popcll(same);
        __syncthreads();
        for (int e = threadIdx.x; e < n_experts; e += threads) {
            int c[16], at = sh.count[0][e];
#pragma unroll
            for (int w = 0; w < 16; ++w) c[w] = w < n_waves ? sh.waves[w * n_experts + e] : 0;
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                if (w < n_waves) sh.waves[w * n_experts + e] = at;
                at += c[w];
            }
            sh.count[0][e] = at;
        }
        __syncthreads();
        if (id >= 0) order[sh.waves[wave * n_experts + id] + rank] = i;
        if (i0 + threads >= hi) break;
        __syncthreads();
        for (int i = threadIdx.x; i < n_waves * n_experts; i += threads) sh.waves[i] = 0;
        __syncthreads();
    }
}

// A workgroup's ids from `per` of them on.
__global__ __launch_bounds__(1024) void moe_plan_kernel(const int32_t *__restrict__ ids, int32_t *__restrict__ starts,
                                                        int32_t *__restrict__ order, int n_experts, int n, int per)
{
    __shared__ PlanShared sh;
    const int lo = blockIdx.x * per;
    plan_range(ids, starts, order, n_experts, n, lo, min(lo + per, n), sh);
}

// One wave a token; lane l holds the experts l, l + 64, ...  Bound by f64 exponentials and divisions where all tokens' waves
// are there at once (4001 tokens, 256 experts, 8 groups: 12.6 to 13.3 us), else by the chain of a token's maxima (one token
// and its plan: 5.6 to 6.1 us; with shuffles of f64 values and a launch of its own for the plan 9.7).  Scores, values and
// their sums are f64, so that the choice does not hang on how a score was rounded.  PLAN: the only workgroup, which goes on
// to the plan.
template <int V, bool PLAN>
__global__ __launch_bounds__(PLAN ? 1024 : 256) void moe_route_kernel(RouteArgs a)
{
    constexpr int kWaves = PLAN ? kOneRoute : 4;
    struct Shared {
        double values[kWaves][V * 64];
        int32_t ids[PLAN ? kWaves * kMaxTopK : 1];
    };
    __shared__ Shared sh;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = blockIdx.x * 4 + wave;
    const double off = -INFINITY;
    if (t < a.batch) {  // no barrier inside: the values are a wave's own
        const float *x = a.logits + (size_t)t * a.n_experts;
        double l[V], score[V];
        float bias[V];
        uint64_t key[V];
        double top = off;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = v * 64 + lane;
            l[v] = e < a.n_experts ? (double)x[e] : off;
            bias[v] = a.bias && e < a.n_experts ? a.bias[e] : 0.0f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) top = l[v] > top ? l[v] : top;
        if (a.scoring == MRML_HIP_MOE_SOFTMAX) {
            // l are f32 values, so their maximum is one of 32 bits
            const uint32_t b = __builtin_bit_cast(uint32_t, (float)top + 0.0f);
            const uint32_t m = wave_max_u32(b >> 31 ? ~b : b | 1u << 31);
            top = (double)__builtin_bit_cast(float, m >> 31 ? m & ~(1u << 31) : ~m);
            double s = 0.0;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                score[v] = !(l[v] > off) ? 0.0 : l[v] == top ? 1.0 : exp(l[v] - top);
                s += score[v];
            }
            s = wave_sum_f64(s);
#pragma unroll
            for (int v = 0; v < V; ++v) score[v] /= s;
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) score[v] = l[v] > off ? 1.0 / (1.0 + exp(-l[v])) : 0.0;
        }
        const bool by_score = a.bias || (a.group_best == 2 && a.n_groups > 1);
#pragma unroll
        for (int v = 0; v < V; ++v)
            key[v] = l[v] > off ? sort_key(by_score ? score[v] + (double)bias[v] : l[v]) : 0;
        if (a.n_groups > 1) {
            // as many lanes a group as there are, a power of two of them: each the two best of its share, then theirs
            const int size = a.n_experts / a.n_groups, shift = 31 - __clz(64 / a.n_groups), g = lane >> shift;
            double *mine = sh.values[wave];
#pragma unroll
            for (int v = 0; v < V; ++v) mine[v * 64 + lane] = key_value(key[v]);
            __builtin_amdgcn_wave_barrier();
            double b1 = off, b2 = off;
            if (g < a.n_groups)
                for (int i = lane & ((1 << shift) - 1); i < size; i += 1 << shift) {
                    const double y = mine[g * size + i];
                    b2 = y > b1 ? b1 : y > b2 ? y : b2;
                    b1 = y > b1 ? y : b1;
                }
            for (int m = 1; m < 1 << shift; m *= 2) {
                const double c1 = __shfl_xor(b1, m, 64), c2 = __shfl_xor(b2, m, 64);
                const double low = c1 > b1 ? b1 : c1;
                b1 = c1 > b1 ? c1 : b1;
                b2 = c2 > b2 ? c2 : b2;
                b2 = low > b2 ? low : b2;
            }
            const double rank = a.group_best == 2 && b2 > off ? b1 + b2 : b1;
            int ahead = 0;  // groups before this one: larger first, equal ones by number
            for (int o = 0; o < a.n_groups; ++o) {
                const double r = lane_f64(rank, o << shift);
                ahead += r > rank || (r == rank && o < g);
            }
            const uint64_t kept = __ballot(ahead < a.top_groups);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int e = v * 64 + lane;
                if (e < a.n_experts && !((kept >> ((e / size) << shift)) & 1)) key[v] = 0;
            }
        }
        int id = -1;  // of slot `lane`
        double got = 0.0;
        for (int s = 0; s < a.k; ++s) {
            uint64_t best = 0;
            double sc = 0.0;
            int e = 1 << 30;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (key[v] > best) {
                    best = key[v];
                    e = v * 64 + lane;
                    sc = score[v];
                }
            const int first = wave_first(best, e);
            if (first < 0) break;
            const int chosen = __builtin_amdgcn_readlane(e, first);
            sc = lane_f64(sc, first);
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v * 64 + lane == chosen) key[v] = 0;
            if (lane == s) {
                id = chosen;
                got = sc;
            }
        }
        const double total = wave_sum_f64(got);
        if (lane < a.k) {
            if (a.renormalise) got = total > 0.0 ? got / total : 0.0;
            a.ids[(size_t)t * a.k + lane] = id;
            a.weights[(size_t)t * a.k + lane] = (float)(got * (double)a.scale);
            if constexpr (PLAN) sh.ids[t * a.k + lane] = id;
        }
    }
    if constexpr (PLAN) {
        __shared__ PlanShared plan;
        __syncthreads();
        plan_range(sh.ids, a.starts, a.order, a.n_experts, a.batch * a.k, 0, a.batch * a.k, plan);
    }
}

}  // namespace

int launch_residual_norm_rows(mrml_hip_ctx *ctx, const float *t, const float *w_post, const float *h, float *h_out,
                              const float *w_next, float *xn, void *pack, int dim, int batch, float eps, bool norm_t)
{
#define NORM_ROWS(CH, THREADS)                                                                                    \
    hipLaunchKernelGGL((residual_norm_rows_kernel<CH, THREADS>), dim3(batch), dim3(threads), 0, ctx->stream, t, w_post, \
                       h, h_out, w_next, xn, (uint8_t *)pack, dim, eps, (int)norm_t)
    const int n4 = dim / 4;
    // a row a CU or fewer: as many threads as there are, which shortens the chain of a thread; more rows: 256, so that
    // several rows overlap.  2816 values, up to 1024 / 256 threads: 1 row 4.6 / 5.4 us, 256 6.9 / 7.7, 512 10.1 / 10.6,
    // 1024 15.3 / 14.4
    if (batch <= 256) {
        const int chunks = (n4 + 1023) / 1024, threads = ((n4 + chunks - 1) / chunks + 63) / 64 * 64;
        if (chunks <= 1) NORM_ROWS(1, 1024);
        else if (chunks <= 2) NORM_ROWS(2, 1024);
        else NORM_ROWS(3, 1024);
    } else {
        const int chunks = (n4 + 255) / 256, threads = 256;
        if (chunks <= 1) NORM_ROWS(1, 256);
        else if (chunks <= 2) NORM_ROWS(2, 256);
        else if (chunks <= 3) NORM_ROWS(3, 256);
        else if (chunks <= 4) NORM_ROWS(4, 256);
        else if (chunks <= 8) NORM_ROWS(8, 256);
        else NORM_ROWS(12, 256);
    }
#undef NORM_ROWS
    return check_launch(ctx, "residual_norm_rows_kernel");
}

int launch_moe_logits(mrml_hip_ctx *ctx, const float *x, const float *w, float *logits, int n_experts, int cols,
                      int batch)
{
    // One wave each / tiles: 128 experts, 16 tokens 5.3 / 6.5 us, 40 5.6 / 6.6, 64 7.0 / 6.7; 32 experts, 64 tokens 4.4 / 6.4.
    // A wave each reads the whole matrix for each token, so the line is late for more experts: 256, 24 tokens 6.0 / 6.6, 40 10.8
    // / 6.7; 512, 4 tokens 5.8 / 6.8, 8 8.3 / 6.9, 40 16.7 / 7.4.
    if (batch <= 40) {
        hipLaunchKernelGGL(moe_logits_kernel, dim3(batch, (n_experts + 3) / 4), dim3(256), 0, ctx->stream, x, w, logits,
                           n_experts, cols, batch);
        return check_launch(ctx, "moe_logits_kernel");
    }
    // a multiple of eight groups of tokens; the rest have none
    auto tiles = [&](int s) { return ((batch + s - 1) / s + 7) / 8 * 8 * ((n_experts + s - 1) / s); };
    const dim3 block(512);
    if (tiles(16) <= 768)
        hipLaunchKernelGGL(moe_logits_tile_kernel<1>, dim3(tiles(16)), block, 0, ctx->stream, x, w, logits, n_experts, cols,
                           batch);
    else
        hipLaunchKernelGGL(moe_logits_tile_kernel<2>, dim3(tiles(32)), block, 0, ctx->stream, x, w, logits, n_experts, cols,
                           batch);
    return check_launch(ctx, "moe_logits_tile_kernel");
}

template <bool PLAN>
static void launch_route(mrml_hip_ctx *ctx, const RouteArgs &a, dim3 grid, dim3 block)
{
    if (a.n_experts <= 64) hipLaunchKernelGGL((moe_route_kernel<1, PLAN>), grid, block, 0, ctx->stream, a);
    else if (a.n_experts <= 128) hipLaunchKernelGGL((moe_route_kernel<2, PLAN>), grid, block, 0, ctx->stream, a);
    else if (a.n_experts <= 256) hipLaunchKernelGGL((moe_route_kernel<4, PLAN>), grid, block, 0, ctx->stream, a);
    else hipLaunchKernelGGL((moe_route_kernel<8, PLAN>), grid, block, 0, ctx->stream, a);
}

int launch_moe_route(mrml_hip_ctx *ctx, const RouteArgs &a)
{
    if (a.starts && a.batch <= kOneRoute) {
        launch_route<true>(ctx, a, dim3(1), dim3(64 * std::max(a.batch, 4)));
        return check_launch(ctx, "moe_route_kernel");
    }
    launch_route<false>(ctx, a, dim3((a.batch + 3) / 4), dim3(256));
    if (int rc = check_launch(ctx, "moe_route_kernel")) return rc;
    if (!a.starts) return MRML_HIP_OK;
    const int n = a.batch * a.k, per = ((n + 255) / 256 + 1023) / 1024 * 1024;
    hipLaunchKernelGGL(moe_plan_kernel, dim3((n + per - 1) / per), dim3(1024), 0, ctx->stream, a.ids, a.starts, a.order,
                       a.n_experts, n, per);
    return check_launch(ctx, "moe_plan_kernel");
}

namespace {

struct Span {
    const void *p;
    size_t bytes;
};

bool overlap(const Span &a, const Span &b)
{
    return a.p && b.p && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes && (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
}

// Whether an output shares memory with another one or with an input.
bool any_overlap(const Span *out, int n_out, const Span *in, int n_in)
{
    for (int i = 0; i < n_out; ++i) {
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return true;
        for (int j = 0; j < n_in; ++j)
            if (overlap(out[i], in[j])) return true;
    }
    return false;
}

bool aligned(uintptr_t bits, uintptr_t to) { return (bits & (to - 1)) == 0; }

int batch_ok(mrml_hip_ctx *ctx, const char *name, int32_t n_experts, int32_t batch, int32_t k)
{
    REQUIRE(ctx, n_experts >= 1 && n_experts <= kMaxExperts, "%s: n_experts=%d (1..%d)", name, n_experts, kMaxExperts);
    REQUIRE(ctx, k >= 1 && k <= kMaxTopK && k <= n_experts, "%s: k=%d (1..%d, at most n_experts=%d)", name, k, kMaxTopK,
            n_experts);
    REQUIRE(ctx, batch >= 1 && (int64_t)batch * k <= kMaxAssignments, "%s: batch=%d of %d experts each (at least one, at "
            "most %d in all)", name, batch, k, kMaxAssignments);
    return MRML_HIP_OK;
}

int product_ok(mrml_hip_ctx *ctx, const char *name, const ExpertArgs &a, bool down)
{
    const float *x = a.x;
    REQUIRE(ctx, a.w[0] && (down || a.w[1]) && (x || a.xpack) && a.ids && a.starts && a.order && a.out &&
                     (!down || a.weights), "%s: null pointer", name);
    if (int rc = batch_ok(ctx, name, a.n_experts, a.batch, a.k)) return rc;
    REQUIRE(ctx, a.cols >= 32 && a.cols % 32 == 0 && a.cols <= kMaxExpertCols, "%s: cols=%d (a multiple of 32 up to %d)",
            name, a.cols, kMaxExpertCols);
    REQUIRE(ctx, a.rows >= 1 && a.rows <= (1 << 20) && (int64_t)a.rows * a.n_experts <= INT32_MAX,
            "%s: rows=%d of %d experts (at least one, at most 2^20, below 2^31 in all)", name, a.rows, a.n_experts);
    REQUIRE(ctx, (int64_t)a.rows * (a.cols / 32) < (1 << 28), "%s: a matrix of %d x %d values has 2^28 blocks or more", name,
            a.rows, a.cols);
    const uintptr_t bits = (uintptr_t)a.w[0] | (uintptr_t)a.w[1] | (uintptr_t)x | (uintptr_t)a.xpack | (uintptr_t)a.out;
    REQUIRE(ctx, aligned(bits, 16), "%s: pointers must be 16-byte aligned", name);
    REQUIRE(ctx, aligned((uintptr_t)a.ids | (uintptr_t)a.starts | (uintptr_t)a.order | (uintptr_t)a.weights, 4),
            "%s: ids, weights, starts and order must be 4-byte aligned", name);
    const size_t n = (size_t)a.batch * a.k, matrix = (size_t)a.n_experts * a.rows * (a.cols / 32) * 18;
    const size_t in_rows = down ? n : a.batch, out_rows = down ? a.batch : n;
    const Span out[] = {{a.out, out_rows * a.rows * 4}};
    const Span in[] = {{a.w[0], matrix}, {a.w[1], matrix}, {x, in_rows * a.cols * 4}, {a.xpack, in_rows * a.cols / 32 * 40},
                       {a.ids, n * 4}, {a.starts, (a.n_experts + 1) * sizeof(int32_t)}, {a.order, n * 4}, {a.weights, n * 4}};
    REQUIRE(ctx, !any_overlap(out, 1, in, 8), "%s: the output shares memory with an input", name);
    return MRML_HIP_OK;
}

}  // namespace

}  // namespace mrml

using namespace mrml;

extern "C" {

int mrml_hip_residual_rms_norm_batch(mrml_hip_ctx *ctx, const float *t, const float *w_post, const float *h,
                                     float *h_out, const float *w_next, float *xn, void *pack, int32_t dim,
                                     int32_t batch, float eps, int32_t norm_t)
{
    CTX_GUARD(ctx);
    const char *name = "residual_rms_norm_batch";
    REQUIRE(ctx, t && h && h_out, "%s: t, h and h_out are required", name);
    REQUIRE(ctx, norm_dim_ok(dim), "%s: dim=%d must be a multiple of 32 up to 12288", name, dim);
    REQUIRE(ctx, batch >= 1 && batch <= (1 << 20), "%s: batch=%d (1..2^20)", name, batch);
    REQUIRE(ctx, aligned((uintptr_t)t | (uintptr_t)w_post | (uintptr_t)h | (uintptr_t)h_out | (uintptr_t)w_next |
                             (uintptr_t)xn | (uintptr_t)pack, 16), "%s: pointers must be 16-byte aligned", name);
    const size_t all = (size_t)batch * dim * 4, one = (size_t)dim * 4;
    const Span out[] = {{h_out, all}, {xn, all}, {pack, all / 128 * 40}};
    // a thread reads its part of a row of t and h before it writes the same part of h_out and xn
    const Span in[] = {{t == xn ? nullptr : t, all}, {h == h_out ? nullptr : h, all}, {norm_t ? w_post : nullptr, one},
                       {w_next, one}};
    REQUIRE(ctx, !any_overlap(out, 3, in, 4), "%s: an output shares memory with another argument (h_out may be h, and xn "
            "may be t)", name);
    return launch_residual_norm_rows(ctx, t, w_post, h, h_out, w_next, xn, pack, dim, batch, eps, norm_t != 0);
}

int mrml_hip_moe_logits(mrml_hip_ctx *ctx, const float *x, const float *w, float *logits, int32_t n_experts,
                        int32_t cols, int32_t batch)
{
    CTX_GUARD(ctx);
    const char *name = "moe_logits";
    REQUIRE(ctx, x && w && logits, "%s: null pointer", name);
    if (int rc = batch_ok(ctx, name, n_experts, batch, 1)) return rc;
    REQUIRE(ctx, cols >= 32 && cols % 32 == 0 && cols <= kMaxExpertCols, "%s: cols=%d (a multiple of 32 up to %d)", name,
            cols, kMaxExpertCols);
    REQUIRE(ctx, aligned((uintptr_t)x | (uintptr_t)w, 16) && aligned((uintptr_t)logits, 4),
            "%s: x and w must be 16-byte aligned, logits 4-byte aligned", name);
    const Span out[] = {{logits, (size_t)batch * n_experts * 4}};
    const Span in[] = {{x, (size_t)batch * cols * 4}, {w, (size_t)n_experts * cols * 4}};
    REQUIRE(ctx, !any_overlap(out, 1, in, 2), "%s: the output shares memory with an input", name);
    return launch_moe_logits(ctx, x, w, logits, n_experts, cols, batch);
}

int mrml_hip_moe_route(mrml_hip_ctx *ctx, const float *logits, const float *bias, int32_t *ids, float *weights,
                       int32_t *starts, int32_t *order, int32_t n_experts, int32_t batch, int32_t k, int32_t scoring,
                       int32_t n_groups, int32_t top_groups, int32_t group_best, int32_t renormalise, float scale)
{
    CTX_GUARD(ctx);
    const char *name = "moe_route";
    REQUIRE(ctx, logits && ids && weights && !starts == !order, "%s: null pointer (starts and order go together)", name);
    if (int rc = batch_ok(ctx, name, n_experts, batch, k)) return rc;
    REQUIRE(ctx, scoring == MRML_HIP_MOE_SOFTMAX || scoring == MRML_HIP_MOE_SIGMOID, "%s: scoring=%d", name, scoring);
    REQUIRE(ctx, n_groups >= 1 && n_groups <= 64 && n_experts % n_groups == 0 && top_groups >= 1 &&
                     top_groups <= n_groups, "%s: n_groups=%d (1..64, a divisor of n_experts=%d), top_groups=%d", name,
            n_groups, n_experts, top_groups);
    REQUIRE(ctx, group_best == 1 || group_best == 2, "%s: group_best=%d (1 or 2)", name, group_best);
    REQUIRE(ctx, std::isfinite(scale), "%s: scale=%g", name, (double)scale);
    REQUIRE(ctx, aligned((uintptr_t)logits | (uintptr_t)bias | (uintptr_t)ids | (uintptr_t)weights | (uintptr_t)starts |
                             (uintptr_t)order, 4), "%s: pointers must be 4-byte aligned", name);
    const size_t n = (size_t)batch * k * 4;
    const Span out[] = {{ids, n}, {weights, n}, {starts, (n_experts + 1) * sizeof(int32_t)}, {order, n}};
    const Span in[] = {{logits, (size_t)batch * n_experts * 4}, {bias, (size_t)n_experts * 4}};
    REQUIRE(ctx, !any_overlap(out, 4, in, 2), "%s: an output shares memory with another argument", name);
    return launch_moe_route(ctx, {logits, bias, ids, weights, starts, order, n_experts, batch, k, scoring, n_groups,
                                  top_groups, group_best, renormalise, scale});
}

static int gate_up(mrml_hip_ctx *ctx, const char *name, const ExpertArgs &a)
{
    if (int rc = product_ok(ctx, name, a, false)) return rc;
    REQUIRE(ctx, a.activation == MRML_HIP_MOE_GEGLU || a.activation == MRML_HIP_MOE_SWIGLU, "%s: activation=%d", name,
            a.activation);
    return launch_moe_gate_up(ctx, a);
}

int mrml_hip_moe_gate_up_q4_0(mrml_hip_ctx *ctx, const void *w_gate, const void *w_up, const float *x,
                              const int32_t *ids, const int32_t *starts, const int32_t *order, float *act,
                              int32_t n_experts, int32_t rows, int32_t cols, int32_t batch, int32_t k,
                              int32_t activation)
{
    CTX_GUARD(ctx);
    return gate_up(ctx, "moe_gate_up_q4_0",
                   {{(const uint8_t *)w_gate, (const uint8_t *)w_up}, x, nullptr, ids, starts, order, nullptr, act, nullptr,
                    ctx->d_moe_faults, n_experts, rows, cols, batch, k, activation});
}

int mrml_hip_moe_gate_up_q4_0_q8(mrml_hip_ctx *ctx, const void *w_gate, const void *w_up, const void *xpack,
                                 const int32_t *ids, const int32_t *starts, const int32_t *order, float *act,
                                 int32_t n_experts, int32_t rows, int32_t cols, int32_t batch, int32_t k,
                                 int32_t activation)
{
    CTX_GUARD(ctx);
    return gate_up(ctx, "moe_gate_up_q4_0_q8",
                   {{(const uint8_t *)w_gate, (const uint8_t *)w_up}, nullptr, (const uint8_t *)xpack, ids, starts, order,
                    nullptr, act, nullptr, ctx->d_moe_faults, n_experts, rows, cols, batch, k, activation});
}

int mrml_hip_moe_down_q4_0(mrml_hip_ctx *ctx, const void *w_down, const float *act, const int32_t *ids,
                           const float *weights, const int32_t *starts, const int32_t *order, float *y,
                           int32_t n_experts, int32_t rows, int32_t cols, int32_t batch, int32_t k)
{
    CTX_GUARD(ctx);
    const ExpertArgs a{{(const uint8_t *)w_down, nullptr}, act, nullptr, ids, starts, order, weights, y, nullptr,
                       ctx->d_moe_faults, n_experts, rows, cols, batch, k, 0};
    if (int rc = product_ok(ctx, "moe_down_q4_0", a, true)) return rc;
    return launch_moe_down(ctx, a);
}

}  // extern "C"
