// moe.h -- what the units of the mixture-of-experts layer share.
#pragma once

#include "device.h"
#include "internal.h"

namespace mrml {

constexpr int kMaxExperts = 512, kMaxTopK = 32, kMaxExpertCols = 32768;
constexpr int kMaxAssignments = 1 << 20;  // batch * k

__device__ __forceinline__ void moe_fault(uint32_t *faults)
{
    __hip_atomic_store(faults, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

struct RouteArgs {
    const float *logits, *bias;
    int32_t *ids;
    float *weights;
    int32_t *starts, *order;
    int n_experts, batch, k, scoring, n_groups, top_groups, group_best, renormalise;
    float scale;
};

// One of the experts' products: gate and up (w[0], w[1]), or down (w[0]).
struct ExpertArgs {
    const uint8_t *w[2];
    const float *x;        // rows to quantise, or
    const uint8_t *xpack;  // their activation pack
    const int32_t *ids, *starts, *order;
    const float *weights;
    float *out;
    uint32_t *faults;
    int n_experts, rows, cols, batch, k, activation;
};

// Whether place j of the order is what a route gives: the assignment of an expert whose run holds j, or -1 behind the
// last run.  True for every j only if ids, starts and order agree.
__device__ __forceinline__ bool plan_ok(const ExpertArgs &a, int j)
{
    const int n = a.batch * a.k, o = a.order[j], end = a.starts[a.n_experts], id = a.ids[j];
    if (id < -1 || id >= a.n_experts || end < 0 || end > n) return false;
    if (j >= end) return o == -1;
    if (o < 0 || o >= n) return false;
    const int e = a.ids[o];
    return e >= 0 && e < a.n_experts && a.starts[e] <= j && j < a.starts[e + 1];
}

int launch_residual_norm_rows(mrml_hip_ctx *ctx, const float *t, const float *w_post, const float *h, float *h_out,
                              const float *w_next, float *xn, void *pack, int dim, int batch, float eps, bool norm_t);
int launch_moe_logits(mrml_hip_ctx *ctx, const float *x, const float *w, float *logits, int n_experts, int cols,
                      int batch);
int launch_moe_route(mrml_hip_ctx *ctx, const RouteArgs &a);
int launch_moe_gate_up(mrml_hip_ctx *ctx, const ExpertArgs &a);
int launch_moe_down(mrml_hip_ctx *ctx, const ExpertArgs &a);

}  // namespace mrml
