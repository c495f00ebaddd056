// attn_paged.hip -- attention of a batch of requests over a paged KV cache
// and a prefix that all of them share.
//
// Row i of request r stands at own position lens[r] - rows(r) + i, behind the
// prefix; it sees the prefix and its request's own positions up to itself,
// the last `window` of them.  out = sum_t p_t v_t with p = softmax over the seen t
// of scale * q . k_t.

#include <algorithm>

#include "paged.h"

namespace mrml {

namespace {

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

// One workgroup a row and head: each wave takes every fourth position with a
// running maximum and sum, lanes over the head's values; the waves' parts are
// joined in LDS.
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedAttn a)
{
    constexpr int E = 8;  // values a lane at most
    __shared__ float s_o[4][512], s_m[4], s_l[4];
    __shared__ int s_seq;
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int hd = a.head_dim, kvh = head / a.group;
    if (tid == 0) {
        int r = -1;
        for (int i = 0; i < a.n_seqs; ++i)
            if (row >= a.row_start[i] && row < a.row_start[i + 1]) {
                r = i;
                break;
            }
        s_seq = r;
    }
    __syncthreads();
    const int r = s_seq;
    if (r < 0) return;
    const int longest = a.table_stride * a.map.page_size, len = min(max(a.lens[r], 0), longest);
    const int at = a.prefix_len + len - (a.row_start[r + 1] - row);  // the row's own place
    const int first = a.window ? max(0, at - a.window + 1) : 0;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    const float *qr = a.q + (size_t)row * a.q_stride + (size_t)head * hd;
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
    for (int t = first + wave; t <= at; t += 4) {
        const bool pre = t < a.prefix_len;
        const int p = pre ? t : t - a.prefix_len, pg = page_of(a.map, p);
        const int id = pre ? a.prefix[pg] : a.table[(size_t)r * a.table_stride + pg];
        if (id < 0 || id >= a.map.n_pages) {
            if (lane == 0) page_fault(a.faults);
            continue;
        }
        const size_t slot = (size_t)id * a.map.page_size + (p - pg * a.map.page_size);
        const uint8_t *kr = a.k + (slot * a.n_kv_heads + kvh) * kv_row_bytes(a.k_fmt, hd);
        const uint8_t *vr = a.v + (slot * a.n_kv_heads + kvh) * kv_row_bytes(a.v_fmt, hd);
        float s = 0.0f;
        for (int e = 0; e < E; ++e)
            if (e * 64 + lane < hd) s = fmaf(q[e], kv_value(kr, a.k_fmt, e * 64 + lane), s);
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x, 64);
        s *= a.scale;
        if (s == -INFINITY) continue;  // no weight
        const float m2 = fmaxf(m, s), f = expf(m - m2), w = expf(s - m2);
        l = l * f + w;
        for (int e = 0; e < E; ++e)
            if (e * 64 + lane < hd) o[e] = o[e] * f + w * kv_value(vr, a.v_fmt, e * 64 + lane);
        m = m2;
    }
    for (int e = 0; e < E; ++e) s_o[wave][e * 64 + lane] = o[e];
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float f[4], sum = 0.0f;
    for (int w = 0; w < 4; ++w) {
        f[w] = s_m[w] > -INFINITY ? expf(s_m[w] - top) : 0.0f;
        sum += s_l[w] * f[w];
    }
    for (int d = tid; d < hd; d += 256) {
        const float x = s_o[0][d] * f[0] + s_o[1][d] * f[1] + s_o[2][d] * f[2] + s_o[3][d] * f[3];
        a.out[((size_t)row * a.n_heads + head) * hd + d] = sum == 0.0f ? 0.0f : x / sum;
    }
}

}  // namespace

size_t paged_attn_scratch_bytes(const PagedAttn &) { return 0; }

int launch_paged_attn(mrml_hip_ctx *ctx, const PagedAttn &a, void *)
{
    hipLaunchKernelGGL(paged_rows_kernel, dim3(a.max_rows, a.n_heads), dim3(256), 0, ctx->stream, a);
    return check_launch(ctx, "paged_rows_kernel");
}

}  // namespace mrml
