// rope.h -- where the RoPE kernels take their angles from.
#pragma once

#include "device.h"
#include "internal.h"

namespace mrml {

// Where a RoPE kernel takes its angles (ops.rs:185-208: theta = pos *
// freq_scale / powf(base, 2i/d) in f32, then cosf and sinf):
//  * table: (cosf, sinf) pairs [n_table][head_dim/2] from the host's libm,
//    for pos < n_table;
//  * else freqs: the powf values per pair from the host's libm, theta formed
//    here and cosf / sinf evaluated with the host libm's algorithm
//    (libm_f32.h), so every position gets the host's bits;
//  * else the same with powf in double precision, rounded once.  The host's
//    powf is not correctly rounded everywhere, so a pair's frequency may then
//    differ from it by one ulp: 6 of 13280 pairs over ten bases and eleven
//    head sizes, none at base 10000.
struct RopeArgs {
    const float *table;
    const float *freqs;
    int n_table;
    float base, freq_scale;
    int fused;  // the host libm's FMA build (host_expf_fused)
};

__host__ inline RopeArgs rope_args(const float *table, int n_table, float base, float freq_scale, const float *freqs)
{
    return RopeArgs{table, freqs, table ? n_table : 0, base, freq_scale, (int)host_expf_fused()};
}

__device__ __forceinline__ void rope_cs(const RopeArgs &r, int pos, int i, int head_dim, float &c, float &s)
{
    if (r.table && pos >= 0 && pos < r.n_table) {
        const float2 cs = reinterpret_cast<const float2 *>(r.table)[(size_t)pos * (head_dim >> 1) + i];
        c = cs.x;
        s = cs.y;
    } else if (r.freqs) {
        const float theta = (float)pos * r.freq_scale / r.freqs[i];
        c = mrml_libm::cosf(theta, r.fused != 0);
        s = mrml_libm::sinf(theta, r.fused != 0);
    } else {
        const float expo = (float)(2 * i) / (float)head_dim;
        const float freq = (float)pow((double)r.base, (double)expo);
        const float theta = (float)pos * r.freq_scale / freq;
        c = mrml_libm::cosf(theta, r.fused != 0);
        s = mrml_libm::sinf(theta, r.fused != 0);
    }
}

}  // namespace mrml
