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
    int32_t *named;  // of down where a sum follows the products: 1 for the assignments that those formed, 0 for the others
    uint32_t *faults;
    int n_experts, rows, cols, batch, k, activation;
};

// ---- ids, starts and order against each other -------------------------------------
// They agree if starts ascend from 0 to at most n = batch * k, every place before the last start names an assignment of the
// expert in whose run it lies, a run's assignments ascend (so none is there twice), and every assignment with an expert has
// a place.  Threads 0 .. n look at one assignment and one place each (plan_ok), a workgroup at the starts (starts_ok); the
// products take what is named, an assignment whose place lies in its own expert's run, and read inside the arrays whatever
// these hold.

// Whether starts that a thread sees are a route's; every thread of a workgroup has to ask.
__device__ __forceinline__ bool starts_ok(const ExpertArgs &a, int thread, int threads)
{
    const int n = a.batch * a.k;
    bool ok = a.starts[0] == 0 && a.starts[a.n_experts] <= n;
    for (int e = thread; e < a.n_experts; e += threads) ok = ok && a.starts[e] <= a.starts[e + 1];
    return ok;
}

// Whether assignment i has a place in its expert's run.
__device__ __forceinline__ bool plan_names(const ExpertArgs &a, int i)
{
    const int n = a.batch * a.k, e = a.ids[i];
    if (e < 0 || e >= a.n_experts) return false;
    int lo = min(max(a.starts[e], 0), n);
    const int end = min(a.starts[e + 1], n);
    for (int hi = max(end, lo); lo < hi;) {
        const int mid = lo + (hi - lo) / 2;
        if (a.order[mid] < i) lo = mid + 1;
        else hi = mid;
    }
    return lo < end && a.order[lo] == i;
}

// The part of the agreement that assignment j and place j show; named: plan_names(a, j).
__device__ __forceinline__ bool plan_ok(const ExpertArgs &a, int j, bool named)
{
    const int n = a.batch * a.k, o = a.order[j], id = a.ids[j];
    if (!named && id != -1) return false;
    if (j >= a.starts[a.n_experts]) return o == -1;
    if (o < 0 || o >= n) return false;
    const int e = a.ids[o];
    if (e < 0 || e >= a.n_experts || j < a.starts[e] || j >= a.starts[e + 1]) return false;
    return j <= max(a.starts[e], 0) || a.order[j - 1] < o;
}

// All of it for a handful of assignments, by one workgroup.
__device__ __forceinline__ void check_few(const ExpertArgs &a, int thread, int threads)
{
    bool ok = starts_ok(a, thread, threads);
    if (thread < a.batch * a.k) ok = ok && plan_ok(a, thread, plan_names(a, thread));
    if (!ok) moe_fault(a.faults);
}

int launch_residual_norm_rows(mrml_hip_ctx *ctx, const float *t, const float *w_post, const float *h, float *h_out,
                              const float *w_next, float *xn, void *pack, int dim, int batch, float eps, bool norm_t);
int launch_moe_logits(mrml_hip_ctx *ctx, const float *x, const float *w, float *logits, int n_experts, int cols,
                      int batch);
int launch_moe_route(mrml_hip_ctx *ctx, const RouteArgs &a);
int launch_moe_gate_up(mrml_hip_ctx *ctx, const ExpertArgs &a);
int launch_moe_down(mrml_hip_ctx *ctx, const ExpertArgs &a);

}  // namespace mrml
