// moe.hip -- a mixture-of-experts layer for a batch of tokens, around the
// experts' products (moe_ffn.hip): the residual's addition and norm, the
// router's logits, the route, and the C ABI of them all.

#include <algorithm>
#include <cmath>

#include "moe.h"
#include "norm_block.h"

namespace mrml {

namespace {

// ---- residual and norm -----------------------------------------------------------

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
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

// One workgroup a row, CH float4 a thread.
template <int CH>
__global__ __launch_bounds__(256) void residual_norm_rows_kernel(const float *t, const float *__restrict__ w_post,
                                                                 const float *h, float *h_out,
                                                                 const float *__restrict__ w_next, float *xn,
                                                                 uint8_t *__restrict__ pack, int dim, float eps,
                                                                 int norm_t)
{
    __shared__ double red[2][4];
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

// One wave a token and expert.
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

// ---- the route -----------------------------------------------------------------------

// Whether (a, i) comes before (b, j): larger first, equal ones by index.
__device__ __forceinline__ bool before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

// One wave a token; lane l holds the experts l, l + 64, ...
template <int V>
__global__ __launch_bounds__(256) void moe_route_kernel(RouteArgs a)
{
    __shared__ double values[4][V * 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = blockIdx.x * 4 + wave;
    if (t >= a.batch) return;  // no barrier below: the values are a wave's own
    const double off = -INFINITY;
    const float *x = a.logits + (size_t)t * a.n_experts;
    double l[V], score[V], value[V];
    bool on[V];
    double top = off;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = v * 64 + lane;
        l[v] = e < a.n_experts ? (double)x[e] : off;
        on[v] = l[v] > off;
        if (on[v]) top = fmax(top, l[v]);
    }
    if (a.scoring == MRML_HIP_MOE_SOFTMAX) {
        for (int m = 32; m >= 1; m >>= 1) top = fmax(top, __shfl_xor(top, m, 64));
        double s = 0.0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            score[v] = !on[v] ? 0.0 : l[v] == top ? 1.0 : exp(l[v] - top);
            s += score[v];
        }
        s = wave_sum_f64(s);
#pragma unroll
        for (int v = 0; v < V; ++v) score[v] /= s;
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) score[v] = on[v] ? 1.0 / (1.0 + exp(-l[v])) : 0.0;
    }
    const bool by_score = a.bias || (a.group_best == 2 && a.n_groups > 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = v * 64 + lane;
        value[v] = by_score ? score[v] + (a.bias && e < a.n_experts ? (double)a.bias[e] : 0.0) : l[v];
        if (!on[v] || !(value[v] > off)) value[v] = off;
    }
    if (a.n_groups > 1) {
        const int size = a.n_experts / a.n_groups;
        double *mine = values[wave];
#pragma unroll
        for (int v = 0; v < V; ++v) mine[v * 64 + lane] = value[v];
        double b1 = off, b2 = off;
        if (lane < a.n_groups)
            for (int i = 0; i < size; ++i) {
                const double y = mine[lane * size + i];
                if (y > b1) {
                    b2 = b1;
                    b1 = y;
                } else if (y > b2) {
                    b2 = y;
                }
            }
        const double rank = a.group_best == 2 && b2 > off ? b1 + b2 : b1;
        int ahead = 0;
        for (int g = 0; g < a.n_groups; ++g) ahead += before(__shfl(rank, g, 64), g, rank, lane);
        const uint64_t kept = __ballot(lane < a.n_groups && ahead < a.top_groups);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = v * 64 + lane;
            if (e < a.n_experts && !((kept >> (e / size)) & 1)) value[v] = off;
        }
    }
    int id = -1;  // of slot `lane`
    double got = 0.0;
    for (int s = 0; s < a.k; ++s) {
        double best = off, sc = 0.0;
        int e = 1 << 30;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (value[v] > best) {
                best = value[v];
                e = v * 64 + lane;
                sc = score[v];
            }
        for (int m = 32; m >= 1; m >>= 1) {
            const double b = __shfl_xor(best, m, 64), o = __shfl_xor(sc, m, 64);
            const int i = __shfl_xor(e, m, 64);
            if (before(b, i, best, e)) {
                best = b;
                e = i;
                sc = o;
            }
        }
        if (!(best > off)) break;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v * 64 + lane == e) value[v] = off;
        if (lane == s) {
            id = e;
            got = sc;
        }
    }
    const double total = wave_sum_f64(got);
    if (lane < a.k) {
        if (a.renormalise) got = total > 0.0 ? got / total : 0.0;
        a.ids[(size_t)t * a.k + lane] = id;
        a.weights[(size_t)t * a.k + lane] = (float)(got * (double)a.scale);
    }
}

// The assignments of expert blockIdx.x in ascending order, behind those of the lower experts; the last workgroup writes
// the end of the list.
__global__ __launch_bounds__(256) void moe_plan_kernel(const int32_t *__restrict__ ids, int32_t *__restrict__ starts,
                                                       int32_t *__restrict__ order, int n_experts, int n)
{
    __shared__ int red[2][4];
    const int e = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int lower = 0;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int id = ids[i];
        lower += id >= 0 && id < e;
    }
    for (int m = 32; m >= 1; m >>= 1) lower += __shfl_xor(lower, m, 64);
    if (lane == 0) red[0][wave] = lower;
    __syncthreads();
    int at = red[0][0] + red[0][1] + red[0][2] + red[0][3];
    if (threadIdx.x == 0) starts[e] = at;
    if (e == n_experts) {
        for (int i = at + threadIdx.x; i < n; i += 256) order[i] = -1;
        return;
    }
    for (int i0 = 0; i0 < n; i0 += 256) {
        const int i = i0 + threadIdx.x;
        const bool mine = i < n && ids[i] == e;
        const uint64_t all = __ballot(mine);
        __syncthreads();
        if (lane == 0) red[1][wave] = __popcll(all);
        __syncthreads();
        int p = at;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) p += red[1][w];
            at += red[1][w];
        }
        if (mine) order[p + __popcll(all & ((1ull << lane) - 1))] = i;
    }
}

}  // namespace

int launch_residual_norm_rows(mrml_hip_ctx *ctx, const float *t, const float *w_post, const float *h, float *h_out,
                              const float *w_next, float *xn, void *pack, int dim, int batch, float eps, bool norm_t)
{
    const int chunks = (dim / 4 + 255) / 256;
#define NORM_ROWS(CH)                                                                                               \
    hipLaunchKernelGGL((residual_norm_rows_kernel<CH>), dim3(batch), dim3(256), 0, ctx->stream, t, w_post, h, h_out, \
                       w_next, xn, (uint8_t *)pack, dim, eps, (int)norm_t)
    if (chunks <= 1) NORM_ROWS(1);
    else if (chunks <= 2) NORM_ROWS(2);
    else if (chunks <= 3) NORM_ROWS(3);
    else if (chunks <= 4) NORM_ROWS(4);
    else if (chunks <= 8) NORM_ROWS(8);
    else NORM_ROWS(12);
#undef NORM_ROWS
    return check_launch(ctx, "residual_norm_rows_kernel");
}

int launch_moe_logits(mrml_hip_ctx *ctx, const float *x, const float *w, float *logits, int n_experts, int cols,
                      int batch)
{
    hipLaunchKernelGGL(moe_logits_kernel, dim3(batch, (n_experts + 3) / 4), dim3(256), 0, ctx->stream, x, w, logits,
                       n_experts, cols, batch);
    return check_launch(ctx, "moe_logits_kernel");
}

int launch_moe_route(mrml_hip_ctx *ctx, const RouteArgs &a)
{
    const dim3 grid((a.batch + 3) / 4), block(256);
    if (a.n_experts <= 64) hipLaunchKernelGGL(moe_route_kernel<1>, grid, block, 0, ctx->stream, a);
    else if (a.n_experts <= 128) hipLaunchKernelGGL(moe_route_kernel<2>, grid, block, 0, ctx->stream, a);
    else if (a.n_experts <= 256) hipLaunchKernelGGL(moe_route_kernel<4>, grid, block, 0, ctx->stream, a);
    else hipLaunchKernelGGL(moe_route_kernel<8>, grid, block, 0, ctx->stream, a);
    if (int rc = check_launch(ctx, "moe_route_kernel")) return rc;
    if (!a.starts) return MRML_HIP_OK;
    hipLaunchKernelGGL(moe_plan_kernel, dim3(a.n_experts + 1), block, 0, ctx->stream, a.ids, a.starts, a.order, a.n_experts,
                       a.batch * a.k);
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
                   {{(const uint8_t *)w_gate, (const uint8_t *)w_up}, x, nullptr, ids, starts, order, nullptr, act,
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
                    nullptr, act, ctx->d_moe_faults, n_experts, rows, cols, batch, k, activation});
}

int mrml_hip_moe_down_q4_0(mrml_hip_ctx *ctx, const void *w_down, const float *act, const int32_t *ids,
                           const float *weights, const int32_t *starts, const int32_t *order, float *y,
                           int32_t n_experts, int32_t rows, int32_t cols, int32_t batch, int32_t k)
{
    CTX_GUARD(ctx);
    const ExpertArgs a{{(const uint8_t *)w_down, nullptr}, act, nullptr, ids, starts, order, weights, y, ctx->d_moe_faults,
                       n_experts, rows, cols, batch, k, 0};
    if (int rc = product_ok(ctx, "moe_down_q4_0", a, true)) return rc;
    return launch_moe_down(ctx, a);
}

}  // extern "C"
