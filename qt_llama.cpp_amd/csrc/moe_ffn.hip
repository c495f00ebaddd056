// moe_ffn.hip -- the experts' products of a mixture-of-experts layer.

#include <algorithm>

#include "moe.h"
#include "exact_sum.h"

namespace mrml {

namespace {

// Row `row` of a Q4_0 matrix with `nblk` blocks in all times block-quantised values (blocks b0.. of an activation pack
// with `total` blocks), over the wave's lanes.
__device__ __forceinline__ float row_dot(const uint8_t *w, size_t nblk, size_t row, int nb, const uint8_t *pack,
                                         size_t total, size_t b0, int lane)
{
    float s = 0.0f;
    for (int b = lane; b < nb; b += 64) {
        const uint4 q = reinterpret_cast<const uint4 *>(w)[row * nb + b];
        const float dw = f16_bits_to_f32(reinterpret_cast<const uint16_t *>(w + nblk * 16)[row * nb + b]);
        const uint4 lo = reinterpret_cast<const uint4 *>(pack)[2 * (b0 + b)];
        const uint4 hi = reinterpret_cast<const uint4 *>(pack)[2 * (b0 + b) + 1];
        const float da = reinterpret_cast<const float *>(pack + total * 32)[b0 + b];
        int n = -8 * reinterpret_cast<const int32_t *>(pack + total * 36)[b0 + b];
        n = sdot4(q.x & kLoNib, lo.x, n);
        n = sdot4(q.y & kLoNib, lo.y, n);
        n = sdot4(q.z & kLoNib, lo.z, n);
        n = sdot4(q.w & kLoNib, lo.w, n);
        n = sdot4((q.x >> 4) & kLoNib, hi.x, n);
        n = sdot4((q.y >> 4) & kLoNib, hi.y, n);
        n = sdot4((q.z >> 4) & kLoNib, hi.z, n);
        n = sdot4((q.w >> 4) & kLoNib, hi.w, n);
        s += (float)n * (dw * da);
    }
    return mrml_xsum::wave_sum_f32(s);
}

__device__ __forceinline__ float silu(float x) { return x / (1.0f + expf(-x)); }

// One wave an assignment and row.
__global__ __launch_bounds__(256) void moe_gate_up_kernel(ExpertArgs a, const uint8_t *pack)
{
    const int as = blockIdx.x, row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, nb = a.cols / 32;
    if (row >= a.rows) return;
    if (row == 0 && !plan_ok(a, as)) moe_fault(a.faults);
    const int e = a.ids[as];
    if (e < 0 || e >= a.n_experts) return;
    const size_t nblk = (size_t)a.n_experts * a.rows * nb, r = (size_t)e * a.rows + row, total = (size_t)a.batch * nb;
    const size_t b0 = (size_t)(as / a.k) * nb;
    const float g = row_dot(a.w[0], nblk, r, nb, pack, total, b0, lane);
    const float u = row_dot(a.w[1], nblk, r, nb, pack, total, b0, lane);
    if (lane == 0) a.out[(size_t)as * a.rows + row] = (a.activation == MRML_HIP_MOE_GEGLU ? gelu_tanh(g) : silu(g)) * u;
}

// One wave a token and row.
__global__ __launch_bounds__(256) void moe_down_kernel(ExpertArgs a, const uint8_t *pack)
{
    const int t = blockIdx.x, row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, nb = a.cols / 32;
    if (row >= a.rows) return;
    const size_t nblk = (size_t)a.n_experts * a.rows * nb, total = (size_t)a.batch * a.k * nb;
    float y = 0.0f;
    for (int s = 0; s < a.k; ++s) {
        const int as = t * a.k + s, e = a.ids[as];
        if (row == 0 && !plan_ok(a, as)) moe_fault(a.faults);
        if (e < 0 || e >= a.n_experts) continue;
        y += a.weights[as] * row_dot(a.w[0], nblk, (size_t)e * a.rows + row, nb, pack, total, (size_t)as * nb, lane);
    }
    if (lane == 0) a.out[(size_t)t * a.rows + row] = y;
}

// The activation pack of n values in the workspace.
int pack_rows(mrml_hip_ctx *ctx, const ExpertArgs &a, size_t n, const uint8_t **pack)
{
    *pack = a.xpack;
    if (a.xpack) return MRML_HIP_OK;
    REQUIRE(ctx, n <= INT32_MAX, "moe: too many activations for one call");
    uint8_t *ws = (uint8_t *)workspace(ctx, act_pack_bytes(n / 32));
    if (!ws) return MRML_HIP_E_ALLOC;
    *pack = ws;
    return launch_quantize_q8_0(ctx, a.x, nullptr, ws, (int32_t)n);
}

}  // namespace

int launch_moe_gate_up(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    const uint8_t *pack;
    if (int rc = pack_rows(ctx, a, (size_t)a.batch * a.cols, &pack)) return rc;
    REQUIRE(ctx, a.rows <= 65535 * 4, "moe: rows=%d", a.rows);
    hipLaunchKernelGGL(moe_gate_up_kernel, dim3(a.batch * a.k, (a.rows + 3) / 4), dim3(256), 0, ctx->stream, a, pack);
    return check_launch(ctx, "moe_gate_up_kernel");
}

int launch_moe_down(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    const uint8_t *pack;
    if (int rc = pack_rows(ctx, a, (size_t)a.batch * a.k * a.cols, &pack)) return rc;
    REQUIRE(ctx, a.rows <= 65535 * 4, "moe: rows=%d", a.rows);
    hipLaunchKernelGGL(moe_down_kernel, dim3(a.batch, (a.rows + 3) / 4), dim3(256), 0, ctx->stream, a, pack);
    return check_launch(ctx, "moe_down_kernel");
}

}  // namespace mrml
