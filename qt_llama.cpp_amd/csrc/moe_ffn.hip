// moe_ffn.hip -- the experts' products of a mixture-of-experts layer.
//
// y[row] = sum over blocks b of dw_b * (sum over the block's 32 of (q - 8) * x),
// with x = da_b * a the Q8_0 values of an activation row.  For few tokens the inner
// sum is one of whole numbers, exact, and takes a conversion, a product of the two
// scales and an FMA behind it.  In the tiles, which vector instructions bound, it
// is two f16 MFMAs whose f32 result only has to be multiplied by dw and added: one
// FMA an output and block.  There q - 8 is a half as it stands, and x, after a power of
// two per row that puts the largest scale at 2^7 .. 2^8, is split into two halves,
// hi + lo.  x has at most 11 + 7 significant bits and lo is a multiple of 2^-24, so
// the split is exact for blocks whose scale is no less than 2^-21 of the row's
// largest; below that x is off by at most 2^-25, 2^-32 of the row's largest scale.  The
// 32 products are exact, their sum may need 11 + 15 bits and is rounded to f32's 24.

#include <algorithm>
#include <type_traits>

#include "any_bytes.h"
#include "moe.h"
#include "exact_sum.h"

namespace mrml {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// ---- activation rows for the MFMA -----------------------------------------------

// A row of nb blocks is nb * 128 bytes: of each block the hi halves (64 bytes), then the lo halves, in the order in
// which a Q4_0 word's nibbles come apart: group g = 0..3 (16 bytes, one lane's operand) has the values 4g, 4g + 2,
// 4g + 1, 4g + 3 and the same + 16.
constexpr int kXBlock = 128;

struct Tile {
    int expert, first, count, pad;  // places first .. first + count of the order
};

constexpr int kTileRows = 16, kTileGroups = 6;  // rows of a group, groups of a tile at most

// Tiles that a call can have.
int max_tiles(const ExpertArgs &a)
{
    const int n = a.batch * a.k;
    return std::min(n, n / (kTileRows * kTileGroups) + std::min(a.n_experts, n));
}

// One workgroup that lists the tiles: tiles[0].expert of them behind tiles[0], none for starts that do not ascend; then one
// thread an assignment that checks the plan (check_wgs workgroups), then WAVES waves a row.  A row of f32 of up to
// WAVES * CH * 256 values is read once and stays in registers; CH = 0 reads it twice.
template <bool PACKED, int WAVES, int CH>
__global__ __launch_bounds__(256) void moe_pack_kernel(ExpertArgs a, int rows, int check_wgs, uint8_t *__restrict__ xp,
                                                       float *__restrict__ xscale, Tile *__restrict__ tiles)
{
    const int nb = a.cols / 32, n = a.batch * a.k;
    if (blockIdx.x == 0) {
        __shared__ int sizes[kTileGroups];
        const int tid = threadIdx.x;
        int groups[2], mine[2], first[2], count[2];
        for (int v = 0; v < 2; ++v) {
            const int e = tid * 2 + v;
            int s0 = 0, s1 = 0;
            if (e < a.n_experts) {
                s0 = min(max(a.starts[e], 0), n);
                s1 = min(max(a.starts[e + 1], s0), n);
            }
            first[v] = s0;
            count[v] = s1 - s0;
            groups[v] = (count[v] + kTileRows - 1) / kTileRows;
            mine[v] = (groups[v] + kTileGroups - 1) / kTileGroups;
        }
        // tiles of each size (in groups, less one), then where they begin: the largest first
        if (tid < kTileGroups) sizes[tid] = 0;
        const bool bad = __syncthreads_or(!starts_ok(a, tid, 256));
        auto each = [&](auto f) {
            for (int v = 0; v < 2; ++v) {
                int from = first[v], left = count[v];
                for (int i = 0; i < mine[v]; ++i) {
                    const int c = min(left, kTileRows * (groups[v] / mine[v] + (i < groups[v] % mine[v])));
                    f(Tile{tid * 2 + v, from, c, 0}, (c - 1) / kTileRows);
                    from += c;
                    left -= c;
                }
            }
        };
        each([&](const Tile &, int size) { atomicAdd(&sizes[size], 1); });
        __syncthreads();
        if (tid == 0) {
            int at = 0;
            for (int k = kTileGroups - 1; k >= 0; --k) {
                const int c = sizes[k];
                sizes[k] = at;
                at += c;
            }
            tiles[0] = {bad ? 0 : at, 0, 0, 0};
        }
        __syncthreads();
        if (bad) return;
        // (equal sizes in any order: no tile's result depends on its place; runs that do not overlap ask for no more than `most`)
        each([&](const Tile &t, int size) {
            const int at = atomicAdd(&sizes[size], 1);
            tiles[1 + at] = t;
        });
        return;
    }
    if ((int)blockIdx.x <= check_wgs) {
        const int j = (blockIdx.x - 1) * 256 + threadIdx.x;
        const bool bad = __syncthreads_or(!starts_ok(a, threadIdx.x, 256));
        if (j >= n) return;
        const bool named = plan_names(a, j);
        if (a.named) a.named[j] = named && !bad;
        if (bad || !plan_ok(a, j, named)) moe_fault(a.faults);
        return;
    }
    constexpr int T = WAVES * 64;  // threads a row
    const int row = (blockIdx.x - 1 - check_wgs) * (256 / T) + threadIdx.x / T, tid = threadIdx.x % T;
    if (row >= rows) return;  // (WAVES = 4: of the whole workgroup)
    const int n4 = a.cols / 4;
    const float4 *x = reinterpret_cast<const float4 *>(a.x + (size_t)row * a.cols);
    const size_t total = (size_t)rows * nb, b0 = (size_t)row * nb;
    const uint32_t *pq = reinterpret_cast<const uint32_t *>(a.xpack);
    const float *pd = reinterpret_cast<const float *>(a.xpack + total * 32);
    float top = 0.0f;
    auto largest = [&](float4 v) {
        top = fmaxf(fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
    };
    float4 held[CH ? CH : 1];
    if (PACKED) {
        for (int b = tid; b < nb; b += T) top = fmaxf(top, pd[b0 + b]);
    } else if (CH) {
#pragma unroll
        for (int i = 0; i < CH; ++i) held[i] = x[min(i * T + tid, n4 - 1)];
#pragma unroll
        for (int i = 0; i < CH; ++i) largest(held[i]);
    } else {
        for (int c = tid; c < n4; c += T) largest(x[c]);
    }
    for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    if (WAVES > 1) {
        __shared__ float tops[4];
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    }
    if (!PACKED) top = f16_bits_to_f32(f32_to_f16_trunc(top / 127.0f));
    // the largest scale becomes 2^7 .. 2^8, so that values stay below 2^15; infinity counts as the largest half
    const int exp = top > 0.0f ? (int)(__builtin_bit_cast(uint32_t, fminf(top, 65504.0f)) >> 23) - 127 - 7 : 0;
    const float down = __builtin_bit_cast(float, (uint32_t)(127 - exp) << 23);
    if (tid == 0) xscale[row] = __builtin_bit_cast(float, (uint32_t)(127 + exp) << 23);
    uint8_t *dst = xp + b0 * kXBlock;
    auto emit = [&](int c, uint32_t q, float d) {
        if (c >= n4) return;
        const int l = c & 7;
        d *= down;
        const float v0 = d * (float)(int8_t)q, v1 = d * (float)(int8_t)(q >> 16), v2 = d * (float)(int8_t)(q >> 8),
                    v3 = d * (float)(int8_t)(q >> 24);
        const half4v hi = {(_Float16)v0, (_Float16)v1, (_Float16)v2, (_Float16)v3};
        const half4v lo = {(_Float16)(v0 - (float)hi.x), (_Float16)(v1 - (float)hi.y), (_Float16)(v2 - (float)hi.z),
                           (_Float16)(v3 - (float)hi.w)};
        uint8_t *p = dst + (size_t)(c >> 3) * kXBlock + (l & 3) * 16 + (l >> 2) * 8;
        *reinterpret_cast<half4v *>(p) = hi;
        *reinterpret_cast<half4v *>(p + 64) = lo;
    };
    auto quantised = [&](int c, float4 v) {
        uint32_t dbits;
        int sum;
        const uint32_t q = q8_0_block8x4(v, dbits, sum);
        emit(c, q, f16_bits_to_f32(dbits));
    };
    if (CH) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i * T < n4) quantised(i * T + tid, held[i]);
    } else {
        for (int c0 = 0; c0 < n4; c0 += T) {
            const int c = c0 + tid, cc = min(c, n4 - 1);
            if (PACKED) emit(c, pq[b0 * 8 + cc], pd[b0 + (cc >> 3)]);
            else quantised(c, x[cc]);
        }
    }
}

// ---- the products -----------------------------------------------------------------

// Halves 2 PART and 2 PART + 1 of the eight q - 8 of a Q4_0 word, in the order of an activation group.  A nibble put under
// the exponent of 1024 is 1024 + q (the high one 1024 + 16 q).  k1024: 0x64006400 in a register of the caller's (a second
// literal would keep the and from being one instruction with the or).
template <int PART>
__device__ __forceinline__ uint32_t nibble_pair(uint32_t w, uint32_t k1024)
{
    const half2v low = {(_Float16)1032.0f, (_Float16)1032.0f}, by = {(_Float16)0.0625f, (_Float16)0.0625f},
                 high = {(_Float16)-72.0f, (_Float16)-72.0f};
    const uint32_t v = PART & 1 ? w >> 8 : w;
    const half2v h = PART < 2 ? __builtin_bit_cast(half2v, (v & 0x000F000Fu) | k1024) - low
                              : __builtin_elementwise_fma(__builtin_bit_cast(half2v, (v & 0x00F000F0u) | k1024), by, high);
    return __builtin_bit_cast(uint32_t, h);
}

// Words w[i] of lane row g (16 lanes) become words w[g] of lane row i: every lane gets its own part of one block after
// the other where it had loaded one block whole.
__device__ __forceinline__ void turn(uint32_t &w0, uint32_t &w1, uint32_t &w2, uint32_t &w3)
{
    auto swap32 = [](uint32_t &a, uint32_t &b) {
        const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
        a = r[0];
        b = r[1];
    };
    auto swap16 = [](uint32_t &a, uint32_t &b) {
        const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        a = r[0];
        b = r[1];
    };
    swap32(w0, w2);
    swap32(w1, w3);
    swap16(w0, w1);
    swap16(w2, w3);
}

// The value of every lane row, in all rows.
__device__ __forceinline__ void spread(uint32_t v, uint32_t (&out)[4])
{
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const auto even = __builtin_amdgcn_permlane32_swap(r[0], r[0], false, false);
    const auto odd = __builtin_amdgcn_permlane32_swap(r[1], r[1], false, false);
    out[0] = even[0];
    out[1] = odd[0];
    out[2] = even[1];
    out[3] = odd[1];
}

// z / (1 + e^-s(z)) with the hardware's exponential and reciprocal (one step each); gelu_tanh is z * sigmoid(2 u).
__device__ __forceinline__ float gated(float g, float u, int activation)
{
    const float s = activation == MRML_HIP_MOE_GEGLU ? 1.5957691216f * __builtin_fmaf(0.044715f * g * g, g, g) : g;
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950409f * s)) * u;
}

constexpr int kWaves = 4;
constexpr int kGroups = 4;  // weight groups of 16 rows a wave
constexpr int kChunk = 4;   // blocks staged at once

// Weight rows of a wave: two groups of gate and the same of up, or four.
template <bool DOWN>
constexpr int wave_rows()
{
    return DOWN ? 64 : 32;
}

// 16 bytes a lane from memory to LDS at `to` + 16 * lane, without registers.  In asm, since the compiler would wait for it
// before any later read of LDS; the reader's loads_barrier waits for it.
__device__ __forceinline__ void load_to_lds(const uint8_t *from, uint32_t to)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(to) : "memory");
}

// A barrier of the workgroup behind this wave's LDS accesses and all its loads but the last LEFT issued.
template <int LEFT>
__device__ __forceinline__ void loads_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

constexpr int kHalf = kChunk / 2;              // blocks of activations in each of two buffers
constexpr int kTilePart = kHalf * kTileGroups * 2048;  // bytes of a buffer: [block][token group][row / 8] 1 KB each

// 16 NT tokens of one expert times the rows of a workgroup.  Lane (g, i): row i of each weight group, and of the
// activations row i of each token group.  A block of a row of activations is one line of 128 bytes; 1 KB has eight rows,
// whose pieces p lie at p ^ row, so that the 16-byte reads of 16 rows meet all banks.  Two blocks of all groups go to one
// buffer while the two in the other are multiplied; a step's weights are on their way for two of those.
//
// Bound by the issue of vector instructions: with two waves a SIMD an MFMA takes 20 cycles, with two FMAs beside it 22, with
// four 31, and there are 4 here, two of them the blocks' FMAs.  So the order is written out, a product of one token group
// beside the additions of the last one and a part of the next block's halves.  (Left to the compiler the two were one after
// the other for the most part.)  1501 tokens, 128 experts of 704 x 2816, eight a token: gate and up 222 us, 429 TFLOP/s; down
// about 122.  With tiles of up to 64 tokens, which take a block's halves apart more often, 13 and 4 us more; with a request
// for each group's scales 21 and 10 more.  AT_ONCE: scales of a row read together, as its blocks' number allows.  Whole
// calls, gate and up of 2816, 2848, 2880, 2912 columns 240, 284, 255, 291 us: odd numbers of blocks have a request a scale,
// and a last step of one or three blocks.
// (pin: a value is formed in its place, which sched_barrier alone does not see to.)
template <class T>
__device__ __forceinline__ void pin(T &x)
{
    asm volatile("" : "+v"(x));
}

template <bool DOWN, int AT_ONCE, int NT>
__device__ __forceinline__ void tile_product(const ExpertArgs &a, const Tile &tile, int chunk_rows, const uint8_t *xp,
                                             uint8_t *lds, const int *s_as, const float *s_scale)
{
    constexpr int kLoadsW = kGroups + 4 / AT_ONCE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
    const int nb = a.cols / 32, r0 = chunk_rows + wave * wave_rows<DOWN>();
    const bool idle = r0 >= a.rows;  // loads for the others, and leaves the SIMD to them
    // the expert's matrices, 32-bit offsets within one
    const size_t first_block = (size_t)tile.expert * a.rows * nb, blocks = (size_t)a.n_experts * a.rows * nb;
    // this wave's share of a buffer: block wave & 1, rows 8 (wave / 2) .. + 8 of every group
    const uint8_t *xrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int as = max(s_as[t * 16 + (wave >> 1) * 8 + (lane >> 3)], 0);
        xrow[t] = xp + (size_t)(DOWN ? as : as / a.k) * nb * kXBlock + ((lane & 7) ^ (lane >> 3)) * 16;
    }
    const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    const uint32_t put = lds_at + ((wave & 1) * kTileGroups * 2 + (wave >> 1)) * 1024;
    auto load_x = [&](int c, int half) {
        const size_t b = (size_t)min(c * kChunk + half * kHalf + (wave & 1), nb - 1) * kXBlock;
#pragma unroll
        for (int t = 0; t < NT; ++t) load_to_lds(xrow[t] + b, __builtin_amdgcn_readfirstlane(put + half * kTilePart + t * 2048));
    };
    uint32_t row_at[kGroups];
#pragma unroll
    for (int q = 0; q < kGroups; ++q) row_at[q] = (uint32_t)min(r0 + (DOWN ? q : q & 1) * 16 + i, a.rows - 1) * nb;
    uint4 wv[kGroups];
    struct __attribute__((packed, aligned(4))) Pair {  // eight bytes from a multiple of four
        uint32_t x, y;
    };
    // quants: of a block of row i of every group; scales: lane row g has the group g's, which saves requests.  AT_ONCE = 1:
    // four loads of 16 bits, which stay apart until the chunk's turn.
    uint32_t sv[AT_ONCE == 1 ? 4 : 2];
    static_assert(kGroups == 4, "a lane row a group");
    const uint8_t *ws = a.w[DOWN ? 0 : g >> 1] + blocks * 16 +
                        (first_block + (uint32_t)min(r0 + (DOWN ? g : g & 1) * 16 + i, a.rows - 1) * nb) * 2;
    // kLoadsW loads whatever c is, for the wait that counts them: places behind the row's last block are clamped, and what
    // was read there is dropped by chunk_scales (a load left out by a branch let that wait pass before the activations
    // were there).
    auto load_w = [&](int c) {
        const uint32_t b = min(c * kChunk + g, nb - 1);
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            const uint8_t *w = a.w[DOWN ? 0 : q >> 1] + first_block * 16;
            uint32_t at_row = row_at[q];
            asm volatile("" : "+v"(at_row));  // addresses are formed here: kept over the loop they cost 16 registers
            // (an offset of less than 2^32 from an address that all lanes share)
            wv[q] = *reinterpret_cast<const uint4 *>(w + (at_row + b) * 16u);
        }
        if constexpr (AT_ONCE == 4) {
            const Pair s = *reinterpret_cast<const Pair *>(ws + min(c * kChunk, nb - kChunk) * 2);
            sv[0] = s.x;
            sv[1] = s.y;
        } else if constexpr (AT_ONCE == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) sv[h] = *reinterpret_cast<const uint32_t *>(ws + min(c * kChunk + h * 2, nb - 2) * 2);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) sv[j] = *reinterpret_cast<const uint16_t *>(ws + min(c * kChunk + j, nb - 1) * 2);
        }
    };
    // Scales of blocks 2 half and 2 half + 1 of chunk c, whose loads were the last; 0 behind the row's last block, where a
    // half has one before it.
    auto chunk_scales = [&](int c, int half) {
        // a row's last two come with the two before
        if constexpr (AT_ONCE == 4) return half == 0 && c * kChunk + 2 != nb ? sv[0] : sv[1];
        else if constexpr (AT_ONCE == 2) return sv[half];
        else return sv[half * 2] | (c * kChunk + half * 2 + 1 < nb ? sv[half * 2 + 1] << 16 : 0u);
    };
    float4v acc[kGroups][NT];
#pragma unroll
    for (int q = 0; q < kGroups; ++q)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[q][t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t k1024 = 0x64006400u;
    asm volatile("" : "+v"(k1024));
    const uint8_t *hi_at = lds + (i >> 3) * 1024 + (i & 7) * 128 + ((g ^ (i & 7)) * 16);
    const uint8_t *lo_at = lds + (i >> 3) * 1024 + (i & 7) * 128 + (((g ^ (i & 7)) ^ 4) * 16);
    const int chunks = (nb + kChunk - 1) / kChunk;
    load_w(0);
    load_x(0, 0);
    for (int c = 0; c < chunks; ++c) {
        uint32_t w[kGroups][4];
        half4v d[kGroups];
        uint32_t scales[2][4];
        spread(chunk_scales(c, 0), scales[0]);
        spread(chunk_scales(c, 1), scales[1]);
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            w[q][0] = wv[q].x;
            w[q][1] = wv[q].y;
            w[q][2] = wv[q].z;
            w[q][3] = wv[q].w;
            turn(w[q][0], w[q][1], w[q][2], w[q][3]);
            d[q] = __builtin_bit_cast(half4v, (uint64_t)scales[1][q] << 32 | scales[0][q]);
            // done before the barrier: a wait for these weights behind it would be one for the loads issued there too
            asm volatile("" : "+v"(w[q][0]), "+v"(w[q][1]), "+v"(w[q][2]), "+v"(w[q][3]), "+v"(d[q]));
        }
        uint4v wh[2][kGroups];  // of blocks j and j + 1
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            // the buffer's loads: before the first half nothing was issued after them, before the second the weights
            if (half == 0) loads_barrier<0>();
            else loads_barrier<kLoadsW>();  // it is whole, and everyone is through with the other one
            if (half == 0) {
                load_x(c, 1);
                load_w(min(c + 1, chunks - 1));  // always, for the count above
            } else if (c + 1 < chunks) {
                load_x(c + 1, 0);
            }
            if (idle || c * kChunk + half * kHalf >= nb) continue;
            half8v x[2][2];
            float4v p[2][kGroups];
            auto read = [&](int to, int step) {
                const int at = half * kTilePart + (step / NT * kTileGroups + step % NT) * 2048;
                x[to][0] = *reinterpret_cast<const half8v *>(hi_at + at);
                x[to][1] = *reinterpret_cast<const half8v *>(lo_at + at);
            };
            auto add = [&](int from, int q, int step) {
                const float dw = (float)d[q][half * kHalf + step / NT];
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    acc[q][step % NT][v] = __builtin_fmaf(p[from][q][v], dw, acc[q][step % NT][v]);
            };
            read(0, 0);
            if (half == 0)
#pragma unroll
                for (int q = 0; q < kGroups; ++q) {
                    wh[0][q].x = nibble_pair<0>(w[q][0], k1024);
                    wh[0][q].y = nibble_pair<1>(w[q][0], k1024);
                    wh[0][q].z = nibble_pair<2>(w[q][0], k1024);
                    wh[0][q].w = nibble_pair<3>(w[q][0], k1024);
                }
#pragma unroll
            for (int step = 0; step < kHalf * NT; ++step) {  // block step / NT, token group step % NT
                const int now = step & 1, t = step % NT, j = half * kHalf + step / NT;
                if (step + 1 < kHalf * NT) read(now ^ 1, step + 1);
                auto weights = [&](int q) { return __builtin_bit_cast(half8v, wh[j & 1][q]); };
#pragma unroll
                for (int q = 0; q < kGroups; ++q) {
                    p[now][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[now][0], weights(q), float4v{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
                    if (step > 0) {
                        add(now ^ 1, q, step - 1);
                        pin(acc[q][(step - 1) % NT]);
                    }
                    pin(p[now][q]);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int q = 0; q < kGroups; ++q) {
                    p[now][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[now][1], weights(q), p[now][q], 0, 0, 0);
                    if (j + 1 < kChunk)
#pragma unroll
                        for (int n = t * kGroups / NT; n < (t + 1) * kGroups / NT; ++n) {
                            if (q == 0) wh[(j + 1) & 1][n].x = nibble_pair<0>(w[n][j + 1], k1024);
                            if (q == 1) wh[(j + 1) & 1][n].y = nibble_pair<1>(w[n][j + 1], k1024);
                            if (q == 2) wh[(j + 1) & 1][n].z = nibble_pair<2>(w[n][j + 1], k1024);
                            if (q == 3) wh[(j + 1) & 1][n].w = nibble_pair<3>(w[n][j + 1], k1024);
                        }
                    if (j + 1 < kChunk)
#pragma unroll
                        for (int n = t * kGroups / NT; n < (t + 1) * kGroups / NT; ++n) pin(wh[(j + 1) & 1][n]);
                    pin(p[now][q]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int q = 0; q < kGroups; ++q) add((kHalf * NT - 1) & 1, q, kHalf * NT - 1);
        }
    }
    // outputs: token row 4g + v of each group, weight row i
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int as = s_as[t * 16 + 4 * g + v];
            if (as < 0) continue;
            const float scale = s_scale[t * 16 + 4 * g + v];
            float *out = a.out + (size_t)as * a.rows;
            if (DOWN) {
#pragma unroll
                for (int q = 0; q < kGroups; ++q)
                    if (r0 + q * 16 + i < a.rows) out[r0 + q * 16 + i] = acc[q][t][v] * scale;
            } else {
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    if (r0 + q * 16 + i < a.rows)
                        out[r0 + q * 16 + i] = gated(acc[q][t][v] * scale, acc[q + 2][t][v] * scale, a.activation);
            }
        }
}

template <bool DOWN, int AT_ONCE>
__global__ __launch_bounds__(64 * kWaves, 2) void moe_tile_kernel(ExpertArgs a, const Tile *__restrict__ tiles,
                                                                  const uint8_t *__restrict__ xp,
                                                                  const float *__restrict__ xscale, int row_wgs)
{
    __shared__ __align__(16) uint8_t lds[2 * kTilePart];
    __shared__ int s_as[kTileGroups * 16];
    __shared__ float s_scale[kTileGroups * 16];
    // Workgroups go to the eight XCDs in turn.  All of a tile go to one, whose L2 then has its activations; the list is by
    // size, the largest first, and dealt back and forth.
    const int xcd = blockIdx.x & 7, turn = (blockIdx.x >> 3) / row_wgs, at = turn * 8 + (turn & 1 ? 7 - xcd : xcd);
    if (at >= tiles[0].expert) return;
    const Tile tile = tiles[1 + at];
    const int n = a.batch * a.k;
    if (threadIdx.x < kTileGroups * 16) {
        const int j = tile.first + (int)threadIdx.x;
        const int o = (int)threadIdx.x < tile.count ? a.order[j] : -1;
        const bool ok = o >= 0 && o < n && a.ids[o] == tile.expert;
        s_as[threadIdx.x] = ok ? o : -1;
        s_scale[threadIdx.x] = ok ? xscale[DOWN ? o : o / a.k] * (DOWN ? a.weights[o] : 1.0f) : 0.0f;
    }
    __syncthreads();
    const int chunk_rows = ((blockIdx.x >> 3) - turn * row_wgs) * kWaves * wave_rows<DOWN>();
    switch ((tile.count + 15) / 16) {
    case 1: tile_product<DOWN, AT_ONCE, 1>(a, tile, chunk_rows, xp, lds, s_as, s_scale); break;
    case 2: tile_product<DOWN, AT_ONCE, 2>(a, tile, chunk_rows, xp, lds, s_as, s_scale); break;
    case 3: tile_product<DOWN, AT_ONCE, 3>(a, tile, chunk_rows, xp, lds, s_as, s_scale); break;
    case 4: tile_product<DOWN, AT_ONCE, 4>(a, tile, chunk_rows, xp, lds, s_as, s_scale); break;
    case 5: tile_product<DOWN, AT_ONCE, 5>(a, tile, chunk_rows, xp, lds, s_as, s_scale); break;
    default: tile_product<DOWN, AT_ONCE, 6>(a, tile, chunk_rows, xp, lds, s_as, s_scale); break;
    }
}

// ---- few tokens an expert -------------------------------------------------------------

// Bound by the stream of weights (40 tokens, eight of 128 experts of 704 x 2816 each: 91 are asked for, 203 MB for gate and
// up in 38 to 46 us): one workgroup for a run of rows and up to 16 tokens of one expert.  The activations come quantised (a
// launch before; every workgroup quantising its own took 10 us of 57 for 40 tokens) and are put in LDS by every workgroup;
// a wave has kUnits runs of 16 rows one after the other, whose weights go from memory to registers kAhead steps ahead and
// without a barrier, 128 bytes of a row at once (a stream of 64 bytes a row reaches 4.9 TB/s here, of 128 bytes 6.1), and
// through 2 KB of LDS of the wave's own to the lanes that need them.  The block sums are int8 MFMA: 16 (q - 8) is a byte
// after one xor, a shift and two ands, half of what a half of it takes, and an int8 activation is a quarter of hi and lo.
// Token t is row 4 (t & 3) + t / 4 of the MFMA, so that a lane's V results are its tokens' and up to 4 V tokens fold V
// values a lane and not four.
constexpr int kStreamBlocks = 128;  // of a row at most: they are all in LDS
constexpr int kStreamTokens = 16;   // a workgroup at most
constexpr int kStep = 8;            // blocks of a row at once
constexpr int kAhead = 4;           // steps; their scales are read kAhead steps at once
constexpr int kStageAhead = 4;      // loads of activations a thread has under way

// Runs of 16 rows of a wave: gate and up of the same rows, or four of down.
template <bool DOWN>
constexpr int stream_units()
{
    return DOWN ? 4 : 2;
}

// Bytes of a block of 4 V tokens in LDS: [group of 8 values][token][8], then 16 to spread the banks.  Scales follow all
// blocks: [run of 4 blocks][token / 4][token & 3][block of the run].  Before them the waves' own parts.
constexpr int stream_block(int v) { return 4 * v * 32 + 16; }
__host__ __device__ constexpr int stream_blocks(int nb) { return (nb + kStep - 1) / kStep * kStep; }
constexpr int kBounce = 16 * kStep * 16;
size_t stream_lds(int nb, int tokens, int part)
{
    return kWaves * part + (size_t)stream_blocks(nb) * (stream_block(tokens / 4) + tokens * 4);
}

// `count` rows of an activation pack of `total` blocks into LDS; scales of 0 behind the last block, up to a whole step.
// loaded() is called once the first loads are under way.
template <int V, class F>
__device__ __forceinline__ void stream_stage(const uint8_t *pack, size_t total, int nb, const int *s_row, int count,
                                             uint8_t *lds, float *scales, F loaded)
{
    const float *pd = reinterpret_cast<const float *>(pack + total * 32);
    auto scale_at = [&](int t, int b) -> float & {
        return scales[(((b / 4) * V + (t >> 2)) * 4 + (t & 3)) * 4 + b % 4];
    };
    const int n2 = nb * 2, all = count * n2;  // halves of blocks
    int t = 0, c = (int)threadIdx.x;
    for (int k0 = 0; k0 < all; k0 += 64 * kWaves * kStageAhead) {
        uint4 q[kStageAhead];
        float d[kStageAhead];
        int tt[kStageAhead], cc[kStageAhead];
#pragma unroll
        for (int k = 0; k < kStageAhead; ++k) {
            for (; c >= n2 && t < count; ++t) c -= n2;
            tt[k] = t;
            cc[k] = t < count ? c : 0;
            const size_t at = (size_t)s_row[t < count ? t : 0] * n2 + cc[k];
            q[k] = reinterpret_cast<const uint4 *>(pack)[at];
            d[k] = pd[at >> 1];
            c += 64 * kWaves;
        }
        if (k0 == 0) loaded();
#pragma unroll
        for (int k = 0; k < kStageAhead; ++k) {
            if (tt[k] >= count) continue;
            const int b = cc[k] >> 1, h = cc[k] & 1;
            Any32 *dst = reinterpret_cast<Any32 *>(lds + b * stream_block(V) + tt[k] * 8 + h * 4);
            dst[0] = q[k].x;
            dst[4 * V * 2] = q[k].y;
            dst[8 * V * 2] = q[k].z;
            dst[12 * V * 2] = q[k].w;
            if (h == 0) scale_at(tt[k], b) = d[k] * 0.0625f;  // the weights' factor of 16
        }
    }
    if ((int)threadIdx.x < 4 * V)
        for (int b = nb; b % kStep; ++b) scale_at(threadIdx.x, b) = 0.0f;
}

typedef int int4v __attribute__((ext_vector_type(4)));

// Eight scales of a row from block b on, read eight, four, two or one at a time as the blocks in a row align them; behind
// the row's last block any.  (One at a time takes registers that the kernel does not have: 16 of gate and up's and 12 of
// down's lie in scratch.)
template <int AT_ONCE>
__device__ __forceinline__ uint4 load_scales(const uint8_t *ws, uint32_t row_at, int b, int nb)
{
    auto at = [&](int i) { return ws + (row_at + min(i, nb - AT_ONCE)) * 2u; };
    auto one = [&](int i) { return *reinterpret_cast<const uint32_t *>(at(i)); };
    auto two = [&](int i) { return *reinterpret_cast<const uint2 *>(at(i)); };
    auto half = [&](int i) {
        return (uint32_t)*reinterpret_cast<const uint16_t *>(at(i)) | (uint32_t)*reinterpret_cast<const uint16_t *>(at(i + 1)) << 16;
    };
    if (AT_ONCE == 8) return *reinterpret_cast<const uint4 *>(at(b));
    if (AT_ONCE == 4) return make_uint4(two(b).x, two(b).y, two(b + 4).x, two(b + 4).y);
    if (AT_ONCE == 2) return make_uint4(one(b), one(b + 2), one(b + 4), one(b + 6));
    return make_uint4(half(b), half(b + 2), half(b + 4), half(b + 6));
}

// Up to 4 V tokens of one expert.
template <bool DOWN, int AT_ONCE, int V>
__device__ __forceinline__ void stream_pass(const ExpertArgs &a, int expert, int count, uint8_t *lds, const int *s_as,
                                            const int *s_row, const float *s_weight)
{
    constexpr int kUnits = stream_units<DOWN>(), kRows = DOWN ? 16 * kUnits : 16;  // rows of a wave
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
    const int nb = a.cols / 32, steps = (nb + kStep - 1) / kStep;
    const int r0 = (blockIdx.x * kWaves + wave) * kRows;
    const int units = r0 >= a.rows ? 0 : DOWN ? min(kUnits, (a.rows - r0 + 15) / 16) : kUnits;
    // the expert's matrices, 32-bit offsets within one
    const size_t first_block = (size_t)expert * a.rows * nb, blocks = (size_t)a.n_experts * a.rows * nb;
    uint8_t *bounce = lds + wave * kBounce;
    lds += kWaves * kBounce;
    float *scales = reinterpret_cast<float *>(lds + stream_blocks(nb) * stream_block(V));
    // row i of the activations is token 4 (i & 3) + i / 4; rows of no token repeat another
    const uint8_t *xa = lds + (g * 4 * V + ((i & 3) < V ? (i & 3) * 4 : 0) + (i >> 2)) * 8;
    const float *sa = scales + g * 4;
    // A step's loads: lane l has block l & 7 of rows l / 8 and 8 + l / 8.  In LDS block b of row r is at b ^ r ^ (r / 8) of
    // the row's eight: both the writes and the reads (word g of one block of row i) go to all banks.
    const int lr = lane >> 3, lb = lane & 7;
    uint4 *put[2];
    const Any32 *get[kStep];
#pragma unroll
    for (int h = 0; h < 2; ++h) put[h] = reinterpret_cast<uint4 *>(bounce) + (h * 8 + lr) * 8 + (lb ^ lr ^ h);
#pragma unroll
    for (int j = 0; j < kStep; ++j)
        get[j] = reinterpret_cast<const Any32 *>(bounce) + (i * 8 + (j ^ (i & 7) ^ (i >> 3))) * 4 + g;
    uint4 wv[kAhead][2], sv;
    // unit u's rows of this lane: of the quants (two), and of the scales
    auto matrix = [&](int u) { return a.w[DOWN ? 0 : u]; };
    auto row_at = [&](int u, int r) { return (uint32_t)min(r0 + (DOWN ? u * 16 : 0) + r, a.rows - 1) * nb; };
    auto load = [&](int k, int u, int c) {
        const uint8_t *w = matrix(u) + first_block * 16;
        const int b = min(c * kStep + lb, nb - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            wv[k][h] = load_stream16(reinterpret_cast<const uint4 *>(w + (row_at(u, h * 8 + lr) + b) * 16u));
    };
    auto load_scale = [&](int u, int c) {  // lane (g, i): of row i, the blocks of step c + g
        sv = load_scales<AT_ONCE>(matrix(u) + blocks * 16 + first_block * 2, row_at(u, i), (c + g) * kStep, nb);
    };
    const size_t total = (size_t)(DOWN ? a.batch * a.k : a.batch) * nb;
    stream_stage<V>(a.xpack, total, nb, s_row, count, lds, scales, [&]() {
        if (units == 0) return;
        load_scale(0, 0);
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k < steps) load(k, 0, k);
    });
    mrml_xsum::lds_barrier();
    float acc[V] = {}, gate[V] = {};
    for (int unit = 0; unit < units; ++unit) {
        for (int c0 = 0; c0 < steps; c0 += kAhead) {
            uint32_t d[4][4];  // scales 2 n and 2 n + 1 of step c0 + k
            {
                uint32_t t[4];
                const uint32_t v[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    spread(v[n], t);
#pragma unroll
                    for (int k = 0; k < 4; ++k) d[k][n] = t[k];
                }
            }
            if (c0 + kAhead < steps) load_scale(unit, c0 + kAhead);
            else if (unit + 1 < units) load_scale(unit + 1, 0);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int c = c0 + k;
                if (c >= steps) break;
                *put[0] = wv[k][0];
                *put[1] = wv[k][1];
                if (c + kAhead < steps) load(k, unit, c + kAhead);
                else if (unit + 1 < units) load(k, unit + 1, k);
                const uint8_t *x = xa + c * kStep * stream_block(V);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float4v s[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) s[v] = *reinterpret_cast<const float4v *>(sa + ((c * 2 + h) * V + v) * 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t y = *get[4 * h + j] ^ 0x88888888u;
                        const uint64_t both = (uint64_t)(y & 0xF0F0F0F0u) << 32 | ((y << 4) & 0xF0F0F0F0u);
                        const int4v p = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                            *reinterpret_cast<const Any64 *>(x + (4 * h + j) * stream_block(V)), (long)both,
                            int4v{0, 0, 0, 0}, 0, 0, 0);
                        const float dw = f16_bits_to_f32(d[k][2 * h + (j >> 1)] >> (j & 1) * 16 & 0xffffu);
#pragma unroll
                        for (int v = 0; v < V; ++v) acc[v] = __builtin_fmaf((float)p[v], dw * s[v][j], acc[v]);
                    }
                }
            }
        }
        // the unit's sums are whole
        const int row = r0 + (DOWN ? unit * 16 : 0) + i;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int t = 4 * v + g;
            if ((DOWN || unit == 1) && t < count && s_as[t] >= 0 && row < a.rows)
                a.out[(size_t)s_as[t] * a.rows + row] = DOWN ? acc[v] * s_weight[t] : gated(gate[v], acc[v], a.activation);
            gate[v] = acc[v];
            acc[v] = 0.0f;
        }
    }
}

// For short rows: the quants of 16 rows lie behind one another in memory, and their scales, so that a wave reads a whole unit
// as it lies and puts it into LDS of its own, one unit ahead.  (In runs of 128 bytes a row, rows of 22 blocks are read across
// lines, and their scales four bytes at once.)
constexpr int kWholeBlocks = 32;  // of a row at most
constexpr int kWholeLoads = kWholeBlocks * 16 / 64;
// LDS of a wave: rows of nb | 1 blocks, which spread over the banks, then the scales as they lie.
__host__ __device__ constexpr int whole_quants(int nb) { return 16 * (nb | 1) * 16; }
__host__ __device__ constexpr int whole_part(int nb) { return whole_quants(nb) + 16 * nb * 2; }

template <bool DOWN, int V>
__device__ __forceinline__ void stream_whole(const ExpertArgs &a, int expert, int count, uint8_t *lds, const int *s_as,
                                             const int *s_row, const float *s_weight)
{
    constexpr int kUnits = stream_units<DOWN>(), kRows = DOWN ? 16 * kUnits : 16;  // rows of a wave
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
    const int nb = a.cols / 32, r0 = (blockIdx.x * kWaves + wave) * kRows;
    const int units = r0 >= a.rows ? 0 : DOWN ? min(kUnits, (a.rows - r0 + 15) / 16) : kUnits;
    const size_t first_block = (size_t)expert * a.rows * nb, blocks = (size_t)a.n_experts * a.rows * nb;
    uint8_t *mine = lds + wave * whole_part(nb), *halves = mine + whole_quants(nb);
    lds += kWaves * whole_part(nb);
    float *scales = reinterpret_cast<float *>(lds + stream_blocks(nb) * stream_block(V));
    const uint8_t *xa = lds + (g * 4 * V + ((i & 3) < V ? (i & 3) * 4 : 0) + (i >> 2)) * 8;  // as in stream_pass
    const float *sa = scales + g * 4;
    const uint8_t *get = mine + i * (nb | 1) * 16 + g * 4, *half_at = halves + i * nb * 2;
    uint32_t put[kWholeLoads];
#pragma unroll
    for (int k = 0; k < kWholeLoads; ++k) {
        const uint32_t q = k * 64 + lane, r = q / (uint32_t)nb;
        put[k] = r < 16 ? (r * (nb | 1) + q - r * nb) * 16 : 0;
    }
    uint4 wv[kWholeLoads], sv;
    auto load = [&](int u) {
        const uint8_t *w = a.w[DOWN ? 0 : u];
        const uint32_t at = (r0 + (DOWN ? u * 16 : 0)) * nb, last = a.rows * nb - 1;  // blocks of the expert
        const uint8_t *quants = w + first_block * 16, *ws = w + blocks * 16 + first_block * 2;
        sv = load_stream16(reinterpret_cast<const uint4 *>(ws) + min(at / 8 + (uint32_t)lane, last / 8));
#pragma unroll
        for (int k = 0; k < kWholeLoads; ++k)
            if (k * 64 < 16 * nb)
                wv[k] = load_stream16(reinterpret_cast<const uint4 *>(quants + min(at + k * 64 + lane, last) * 16u));
    };
    const size_t total = (size_t)(DOWN ? a.batch * a.k : a.batch) * nb;
    stream_stage<V>(a.xpack, total, nb, s_row, count, lds, scales, [&]() {
        if (units) load(0);
    });
    mrml_xsum::lds_barrier();
    float acc[V] = {}, gate[V] = {};
    for (int unit = 0; unit < units; ++unit) {
#pragma unroll
        for (int k = 0; k < kWholeLoads; ++k)
            if (k * 64 + lane < 16 * nb) *reinterpret_cast<uint4 *>(mine + put[k]) = wv[k];
        if (lane < 2 * nb) reinterpret_cast<uint4 *>(halves)[lane] = sv;
        __builtin_amdgcn_wave_barrier();
        if (unit + 1 < units) load(unit + 1);
        auto block = [&](int b, const float4v (&s)[V], int j) {
            const uint32_t y = *reinterpret_cast<const Any32 *>(get + (b + j) * 16) ^ 0x88888888u;
            const uint64_t both = (uint64_t)(y & 0xF0F0F0F0u) << 32 | ((y << 4) & 0xF0F0F0F0u);
            const int4v p = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                *reinterpret_cast<const Any64 *>(xa + (b + j) * stream_block(V)), (long)both, int4v{0, 0, 0, 0}, 0, 0, 0);
            const float dw = f16_bits_to_f32(*reinterpret_cast<const Any16 *>(half_at + (b + j) * 2));
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = __builtin_fmaf((float)p[v], dw * s[v][j], acc[v]);
        };
        int b = 0;
        for (; b + 4 <= nb; b += 4) {
            float4v s[V];
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = *reinterpret_cast<const float4v *>(sa + (b / 4 * V + v) * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) block(b, s, j);
        }
        if (b < nb) {
            float4v s[V];
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = *reinterpret_cast<const float4v *>(sa + (b / 4 * V + v) * 16);
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (b + j < nb) block(b, s, j);
        }
        __builtin_amdgcn_wave_barrier();
        const int row = r0 + (DOWN ? unit * 16 : 0) + i;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int t = 4 * v + g;
            if ((DOWN || unit == 1) && t < count && s_as[t] >= 0 && row < a.rows)
                a.out[(size_t)s_as[t] * a.rows + row] = DOWN ? acc[v] * s_weight[t] : gated(gate[v], acc[v], a.activation);
            gate[v] = acc[v];
            acc[v] = 0.0f;
        }
    }
}

// Workgroup (x, y): rows of chunk x, and tile y of all experts' tiles of `tokens` tokens.  AT_ONCE = 0: by whole units.
template <bool DOWN, int AT_ONCE>
__global__ __launch_bounds__(64 * kWaves, 4) void moe_stream_kernel(ExpertArgs a, int tokens)
{
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int s_as[kStreamTokens], s_row[kStreamTokens], s_tile[3], s_ends[kWaves], s_bad[kWaves];
    __shared__ float s_weight[kStreamTokens];
    const int n = a.batch * a.k, tid = threadIdx.x;
    // The assignment and place that this thread looks at, from the last workgroup on, as the last ones mostly have no tile.
    // (In 64 bits: 2^24 workgroups are within the limits.)
    const uint64_t j = ((uint64_t)(gridDim.y - 1 - blockIdx.y) * gridDim.x + blockIdx.x) * (64 * kWaves) + tid;
    if (tid == 0) s_tile[2] = 0;
    // tiles of the experts of each thread, and before them
    static_assert(kMaxExperts == 2 * 64 * kWaves, "two experts a thread");
    int first[2], count[2], mine = 0;
    bool ok = a.starts[0] == 0;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int e = 2 * tid + v;
        const int r0 = e < a.n_experts ? a.starts[e] : 0, r1 = e < a.n_experts ? a.starts[e + 1] : 0;
        ok = ok && r0 <= r1 && r1 <= n;
        const int s0 = min(max(r0, 0), n), s1 = min(max(r1, s0), n);
        first[v] = s0;
        count[v] = s1 - s0;
        mine += (count[v] + tokens - 1) / tokens;
    }
    int ends = mine;
    for (int m = 1; m < 64; m *= 2) {
        const int before = __shfl_up(ends, m, 64);
        if ((tid & 63) >= m) ends += before;
    }
    const bool wave_bad = __any(!ok);
    if ((tid & 63) == 63) {
        s_ends[tid >> 6] = ends;
        s_bad[tid >> 6] = wave_bad;
    }
    mrml_xsum::lds_barrier();
    // starts that do not ascend from 0 to at most n: everything is left out
    const bool bad = s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
    int at = ends - mine;
    for (int w = 0; w < (tid >> 6); ++w) at += s_ends[w];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int tiles = (count[v] + tokens - 1) / tokens, t = (int)blockIdx.y - at;
        if (!bad && t >= 0 && t < tiles) {
            s_tile[0] = 2 * tid + v;
            s_tile[1] = first[v] + t * tokens;
            s_tile[2] = min(tokens, count[v] - t * tokens);
        }
        at += tiles;
    }
    mrml_xsum::lds_barrier();
    if (j < (uint32_t)n) {
        const bool named = plan_names(a, (int)j);
        if (DOWN) a.named[j] = named && !bad;
        if (bad || !plan_ok(a, (int)j, named)) moe_fault(a.faults);
    }
    const int e = __builtin_amdgcn_readfirstlane(s_tile[0]), from = __builtin_amdgcn_readfirstlane(s_tile[1]);
    const int tokens_here = __builtin_amdgcn_readfirstlane(s_tile[2]);
    if (tokens_here == 0) return;
    if (tid < kStreamTokens) {
        const int o = tid < tokens_here ? a.order[from + tid] : -1;
        const bool there = o >= 0 && o < n && a.ids[o] == e;
        s_as[tid] = there ? o : -1;
        s_row[tid] = there ? (DOWN ? o : o / a.k) : 0;
        s_weight[tid] = DOWN && there ? a.weights[o] : 0.0f;
    }
    mrml_xsum::lds_barrier();
#define PASS(V)                                                                                          \
    if constexpr (AT_ONCE == 0) stream_whole<DOWN, V>(a, e, tokens_here, lds, s_as, s_row, s_weight);     \
    else stream_pass<DOWN, AT_ONCE, V>(a, e, tokens_here, lds, s_as, s_row, s_weight)
    if (tokens_here <= 4) PASS(1);
    else if (tokens_here <= 8) PASS(2);
    else PASS(4);
#undef PASS
}

// ---- a handful of assignments ------------------------------------------------------------

// Each assignment that is named (moe.h) by itself, in one launch, from the activations as they come (a launch to quantise
// and one for the lists would take as long as the products).  The block sums are the matvecs' (v_dot8 on raw weight words
// and split-nibble activations): lane (r, b) = (lane / 8, lane % 8) has block 8 c + b of row r of 8 in step c, a load of
// 128 bytes a row.
//  A unit's scales are read as one run of memory into LDS of the wave's own (read where they are needed they
// are as many requests as the weights).  What it comes to is a few microseconds of latencies one after the other and the
// rate at which a CU takes loads, so:
//  - units are small, since the CU with the most of them sets the time (eight assignments of 704 rows and 2816 columns:
//    352 workgroups of 16 rows, two on some CUs and one on others, 9.4 us; 704 of 8 rows, three or two, see below);
//  - waves of their own quantise: a CU takes 1.5 to 4 us to accept the loads of its weights, and a wave that issues those
//    first cannot quantise meanwhile.
// A trip to memory stands before the weights' loads all the same: the compiler keeps the first piece of a unit's scales
// (DotUnit::sv) in scratch, 32 bytes a lane, and waits for it before it goes on; down's kernel waits for the activations with it.
constexpr int kGateRows = 8, kDownRows = 16;  // of a workgroup

__host__ __device__ constexpr size_t dot_scales_bytes(int nb, int rows) { return (size_t)nb * rows * 2; }  // of a wave
__host__ __device__ constexpr size_t dot_token_bytes(int nb) { return ((size_t)nb * 40 + 15) / 16 * 16; }

// A token's blocks in LDS: lo and hi (device.h), then behind all blocks {d, c}.
struct DotToken {
    uint4 *x;
    float2 *dc;
    __device__ DotToken(uint8_t *lds, int nb) : x(reinterpret_cast<uint4 *>(lds)), dc(reinterpret_cast<float2 *>(lds + nb * 32)) {}
};

// Block b from its 32 quants.
__device__ __forceinline__ void dot_put(const DotToken &t, int b, uint4 x, uint4 y, float d)
{
    t.x[2 * b] = make_uint4(split_lo(x.x, y.x), split_lo(x.y, y.y), split_lo(x.z, y.z), split_lo(x.w, y.w));
    t.x[2 * b + 1] = make_uint4(split_hi(x.x, y.x), split_hi(x.y, y.y), split_hi(x.z, y.z), split_hi(x.w, y.w));
    const int c = -8 * (lo_nib_sum(x.x) + lo_nib_sum(x.y) + lo_nib_sum(x.z) + lo_nib_sum(x.w) + lo_nib_sum(y.x) +
                        lo_nib_sum(y.y) + lo_nib_sum(y.z) + lo_nib_sum(y.w));
    t.dc[b] = make_float2(d, __builtin_bit_cast(float, c));
}

// A row of f32 quantised by `threads` threads (whole waves), this one `tid`; ahead() once the first loads are under way.
template <class F>
__device__ __forceinline__ void dot_quantize(const float *x, int nb, int tid, int threads, const DotToken &t, F ahead)
{
    constexpr int kBatch = 4;
    const int n4 = nb * 8;
    for (int c0 = 0; c0 < n4; c0 += kBatch * threads) {
        float4 v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) v[k] = reinterpret_cast<const float4 *>(x)[min(c0 + k * threads + tid, n4 - 1)];
        if (c0 == 0) ahead();
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (c0 + k * threads >= n4) break;
            const int c = c0 + k * threads + tid, l = c & 7;
            uint32_t dbits;
            int sum;
            const uint32_t q = q8_0_block8x4(v[k], dbits, sum);
            const uint32_t w = q8_split8(q, l, sum);
            if (c < n4) {
                reinterpret_cast<Any32 *>(t.x)[c] = w;
                if (l == 0) t.dc[c >> 3] = make_float2(f16_bits_to_f32(dbits), __builtin_bit_cast(float, sum));
            }
        }
    }
}

// A unit's 8 H rows of an expert's matrix, and what a wave has of them.
template <int H>
struct DotUnit {
    static constexpr int kScales = kStreamBlocks * H / 64;  // pieces of 16 bytes a lane
    const uint8_t *w, *ws;  // the expert's quants and scales
    uint32_t row, rows;     // first row; rows of the matrix
    uint4 sv[kScales];
    uint4 st[kAhead][H];
    bool wide;

    __device__ __forceinline__ DotUnit(const ExpertArgs &a, int matrix, int expert, int r, int nb) : row(r), rows(a.rows)
    {
        const size_t first = (size_t)expert * a.rows * nb, all = (size_t)a.n_experts * a.rows * nb;
        w = a.w[matrix] + first * 16;
        ws = a.w[matrix] + all * 16 + first * 2;
    }

    __device__ __forceinline__ int halves(int nb) const { return min(8 * H, (int)(rows - row)) * nb; }

    // Scales from memory to registers, 16 bytes a lane, where they lie so; on to LDS.  Rows past the matrix's last get
    // some scales of it.
    __device__ __forceinline__ void load_scales(int nb, int lane)
    {
        const uint8_t *src = ws + (size_t)row * nb * 2;
        wide = (((uintptr_t)src | (uintptr_t)(halves(nb) * 2)) & 15) == 0;
        if (!wide) return;
#pragma unroll
        for (int k = 0; k < kScales; ++k)
            if (k * 64 < nb * H) sv[k] = reinterpret_cast<const uint4 *>(src)[min(k * 64 + lane, halves(nb) / 8 - 1)];
    }
    __device__ __forceinline__ void store_scales(int nb, int lane, Any16 *lds) const
    {
        if (wide) {
#pragma unroll
            for (int k = 0; k < kScales; ++k)
                if (k * 64 + lane < nb * H) reinterpret_cast<uint4 *>(lds)[k * 64 + lane] = sv[k];
        } else {
            const uint16_t *src = reinterpret_cast<const uint16_t *>(ws) + (size_t)row * nb;
            for (int k = lane; k < 8 * H * nb; k += 64) lds[k] = src[min(k, halves(nb) - 1)];
        }
    }

    __device__ __forceinline__ void load(int k, int nb, int c, int lane)
    {
        const int b = min(c * kStep + (lane & 7), nb - 1);
#pragma unroll
        for (int h = 0; h < H; ++h)
            st[k][h] = load_stream16(
                reinterpret_cast<const uint4 *>(w + (min(row + h * 8 + (lane >> 3), rows - 1) * nb + b) * 16ull));
    }

    // Steps c0 .. c1, whose first kAhead are on the way: the sums of rows lane / 8 + 8 h, in all lanes of a row.
    __device__ __forceinline__ void sum(int nb, int c0, int c1, int lane, const Any16 *scales, const DotToken &x,
                                        float (&acc)[H])
    {
#pragma unroll
        for (int h = 0; h < H; ++h) acc[h] = 0.0f;
        for (int s0 = c0; s0 < c1; s0 += kAhead)
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int c = s0 + k, bt = c * kStep + (lane & 7), b = min(bt, nb - 1);
                if (c >= c1) break;
                uint4 q[H];
#pragma unroll
                for (int h = 0; h < H; ++h) q[h] = st[k][h];
                if (c + kAhead < c1) load(k, nb, c + kAhead, lane);
                const uint4 lo = x.x[2 * b], hi = x.x[2 * b + 1];
                const float2 dc = x.dc[b];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const float dw = f16_bits_to_f32(scales[(h * 8 + (lane >> 3)) * nb + b]);
                    const int n = q4_0_isum_split(q[h].x, q[h].y, q[h].z, q[h].w, lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z,
                                                  hi.w, __builtin_bit_cast(int, dc.y));
                    acc[h] = __builtin_fmaf((float)n, (bt < nb ? dw : 0.0f) * dc.x, acc[h]);
                }
            }
        auto from = [](float v, auto ctrl) {
            return __builtin_bit_cast(float, dpp_mov<decltype(ctrl)::value>(__builtin_bit_cast(int, v)));
        };
#pragma unroll
        for (int h = 0; h < H; ++h) {
            acc[h] += from(acc[h], std::integral_constant<int, 0xB1>{});
            acc[h] += from(acc[h], std::integral_constant<int, 0x4E>{});
            acc[h] += from(acc[h], std::integral_constant<int, 0x141>{});
        }
    }
};

// Whether an assignment of expert e is named, of a handful: asked for early, answered at the end.
struct Named {
    int place = -1, lo = 0, hi = 0;
    __device__ __forceinline__ void ask(const ExpertArgs &a, int e, int lane)
    {
        if (lane < a.batch * a.k) place = a.order[lane];
        lo = a.starts[e];
        hi = a.starts[e + 1];
    }
    __device__ __forceinline__ bool yes(int as, int lane) const { return __any(place == as && lane >= lo && lane < hi); }
};

// One assignment (blockIdx.y) and 8 rows of gate and of up, each by two waves that have half of the blocks; four waves more
// quantise the token.
constexpr int kPutWaves = 4, kGetWaves = 4;
__global__ __launch_bounds__(64 * (kPutWaves + kGetWaves)) void moe_gate_up_one_kernel(ExpertArgs a)
{
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ float part[kGetWaves][kGateRows];
    __shared__ int s_named;
    const int tid = threadIdx.x, lane = tid & 63, nb = a.cols / 32, as = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), row0 = blockIdx.x * kGateRows;
    const DotToken token(lds, nb);
    const int e = a.ids[as];
    const bool there = e >= 0 && e < a.n_experts;
    if (wave < kPutWaves) {
        const size_t t = as / a.k;
        if (a.xpack) {
            const uint4 *q = reinterpret_cast<const uint4 *>(a.xpack + t * nb * 32);
            const float *d = reinterpret_cast<const float *>(a.xpack + (size_t)a.batch * nb * 32) + t * nb;
            for (int b = tid; b < nb; b += 64 * kPutWaves) dot_put(token, b, q[2 * b], q[2 * b + 1], d[b]);
        } else {
            dot_quantize(a.x + t * a.cols, nb, tid, 64 * kPutWaves, token, []() {});
        }
        mrml_xsum::lds_barrier();
        if (wave == 0) {  // while the others sum
            Named named;
            if (there) named.ask(a, e, lane);
            const bool yes = named.yes(as, lane);
            if (lane == 0) s_named = yes;
        }
        mrml_xsum::lds_barrier();
        if (blockIdx.x + blockIdx.y == 0) check_few(a, tid, 64 * kPutWaves);
        return;
    }
    const int w = wave - kPutWaves;
    const int steps = there ? (nb + kStep - 1) / kStep : 0, half = (steps + 1) / 2;
    const int c0 = (w & 1) * half, c1 = min(c0 + half, steps);
    Any16 *scales = reinterpret_cast<Any16 *>(lds + dot_token_bytes(nb) + w * dot_scales_bytes(nb, kGateRows));
    DotUnit<1> unit(a, w >> 1, there ? e : 0, row0, nb);
    if (c0 < c1) unit.load_scales(nb, lane);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (c0 + k < c1) unit.load(k, nb, c0 + k, lane);
    if (c0 < c1) unit.store_scales(nb, lane, scales);
    mrml_xsum::lds_barrier();
    float v[1];
    unit.sum(nb, c0, c1, lane, scales, token, v);
    if ((lane & 7) == 0) part[w][lane >> 3] = v[0];
    mrml_xsum::lds_barrier();
    const int r = tid - 64 * kPutWaves;
    if (r < kGateRows && row0 + r < a.rows && s_named)
        a.out[(size_t)as * a.rows + row0 + r] = gated(part[0][r] + part[1][r], part[2][r] + part[3][r], a.activation);
}

// One token (blockIdx.y) and 16 rows of down, eight of its assignments at a time, a wave each, which quantises it; y itself.
constexpr int kDownWaves = 8;
__global__ __launch_bounds__(64 * kDownWaves) void moe_down_one_kernel(ExpertArgs a)
{
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ float part[kMaxTopK][kDownRows];
    const int tid = threadIdx.x, lane = tid & 63, nb = a.cols / 32, t = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row0 = blockIdx.x * kDownRows, steps = (nb + kStep - 1) / kStep;
    uint8_t *mine = lds + wave * (dot_token_bytes(nb) + dot_scales_bytes(nb, kDownRows));
    const DotToken token(mine, nb);
    // No token: the first of these checks the plan.  (Behind the rows of a workgroup that has some it takes 0.8 us of a
    // call.  In a column of its own it leaves the tokens' workgroups for one row run on different XCDs, which read the
    // weights again: eight tokens, four experts, two a token 22.5 us, so 20.2.)
    if (t == a.batch) {
        if (blockIdx.x == 0) check_few(a, tid, 64 * kDownWaves);
        return;
    }
    Any16 *scales = reinterpret_cast<Any16 *>(mine + dot_token_bytes(nb));
    for (int s = wave; s < a.k; s += kDownWaves) {
        const int as = t * a.k + s, e = a.ids[as];
        const bool there = e >= 0 && e < a.n_experts;
        const float weight = there ? a.weights[as] : 0.0f;
        Named named;
        float v[2] = {0.0f, 0.0f};
        if (there) {
            named.ask(a, e, lane);
            DotUnit<2> unit(a, 0, e, row0, nb);
            dot_quantize(a.x + (size_t)as * a.cols, nb, lane, 64, token, [&]() {
                unit.load_scales(nb, lane);
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
                    if (k < steps) unit.load(k, nb, k, lane);
            });
            unit.store_scales(nb, lane, scales);
            unit.sum(nb, 0, steps, lane, scales, token, v);
        }
        const bool in = named.yes(as, lane);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if ((lane & 7) == 0) part[s][h * 8 + (lane >> 3)] = in ? v[h] * weight : 0.0f;
    }
    mrml_xsum::lds_barrier();
    if (tid < kDownRows && row0 + tid < a.rows) {
        float y = 0.0f;
        for (int s = 0; s < a.k; ++s) y += part[s][tid];
        a.out[(size_t)t * a.rows + row0 + tid] = y;
    }
}

// y = the sum of a token's weighted products (a.out) in the order of its slots, of those that were formed (a.named); VEC
// values a thread, eight slots' loads at once.  Bound by its bytes: 1501 tokens of eight slots, 2816 rows: 24 us for 152
// MB, some of them still in a cache.
template <int VEC>
__global__ __launch_bounds__(256) void moe_combine_kernel(ExpertArgs a, float *__restrict__ y)
{
    const int t = blockIdx.x, r = (blockIdx.y * 256 + threadIdx.x) * VEC;
    if (r >= a.rows) return;
    typedef float vec __attribute__((ext_vector_type(VEC)));
    vec s = 0.0f;
    for (int i0 = 0; i0 < a.k; i0 += 8) {
        vec v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int as = t * a.k + min(i0 + i, a.k - 1);
            v[i] = 0.0f;
            if (i0 + i < a.k && a.named[as]) v[i] = *reinterpret_cast<const vec *>(a.out + (size_t)as * a.rows + r);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
    }
    *reinterpret_cast<vec *>(y + (size_t)t * a.rows + r) = s;
}

template <bool DOWN>
int row_wgs(const ExpertArgs &a)  // workgroups of a tile
{
    return (a.rows + kWaves * wave_rows<DOWN>() - 1) / (kWaves * wave_rows<DOWN>());
}

template <bool DOWN>
int64_t tile_grid(const ExpertArgs &a, int most)
{
    return (int64_t)(most + 7) / 8 * 8 * row_wgs<DOWN>(a);
}

template <bool DOWN>
int launch_tiles(mrml_hip_ctx *ctx, const ExpertArgs &a, int most, const Tile *tiles, const uint8_t *xp, const float *xscale)
{
    const int64_t grid = tile_grid<DOWN>(a, most);
    const int nb = a.cols / 32;
#define TILES(AT_ONCE)                                                                                                \
    hipLaunchKernelGGL((moe_tile_kernel<DOWN, AT_ONCE>), dim3((uint32_t)grid), dim3(64 * kWaves), 0, ctx->stream, a, tiles, \
                       xp, xscale, row_wgs<DOWN>(a))
    if (nb % 2 == 0 && nb >= kChunk) TILES(4);
    else if (nb % 2 == 0) TILES(2);
    else TILES(1);
#undef TILES
    return check_launch(ctx, "moe_tile_kernel");
}

// A handful of assignments: each by itself, from the activations as they come.  So / streamed or in tiles, experts of 704 x
// 2816 (down: 2816 x 704), in us: 128 experts, eight a token, 1, 2, 3 tokens: gate and up 7.0 / 17.4, 11.3 / 17.6, 15.1 / 17.9,
// down 6.7 / 15.9, 12.0 / 15.9, 17.7 / 16.0; eight experts, two a token, 4, 8, 12 tokens: gate and up 6.6 / 17.2, 10.1 /
// 17.9, 13.5 / 19.9, down 11.3 / 15.1, 21.2 / 16.0, 33.0 / 17.6.  The line looks at the number of assignments alone.  It is
// late where an expert's matrices are read once for each of several tokens and take longer than the other forms' launches:
// down of one expert, 4, 8, 16 tokens 10.3 / 15.4, 19.1 / 15.5, 34.7 / 15.7; gate and up of 14336 x 4096, eight experts,
// two a token, 1, 4, 8 tokens 29.8 / 27.8, 107 / 60, 208 / 83.
bool one_by_one(const ExpertArgs &a) { return a.batch * a.k <= 16 && a.cols / 32 <= kStreamBlocks; }

int launch_gate_up_one(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    const int nb = a.cols / 32;
    const size_t lds = dot_token_bytes(nb) + kGetWaves * dot_scales_bytes(nb, kGateRows);
    hipLaunchKernelGGL(moe_gate_up_one_kernel, dim3((a.rows + kGateRows - 1) / kGateRows, a.batch * a.k),
                       dim3(64 * (kPutWaves + kGetWaves)), lds, ctx->stream, a);
    return check_launch(ctx, "moe_gate_up_one_kernel");
}

int launch_down_one(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    const int nb = a.cols / 32;
    const size_t lds = kDownWaves * (dot_token_bytes(nb) + dot_scales_bytes(nb, kDownRows));
    hipLaunchKernelGGL(moe_down_one_kernel, dim3((a.rows + kDownRows - 1) / kDownRows, a.batch + 1), dim3(64 * kDownWaves), lds,
                       ctx->stream, a);
    return check_launch(ctx, "moe_down_one_kernel");
}

// Few tokens an expert on average, or, for gate and up, so few tiles that they would leave CUs without any, where a pass over
// the weights for every 16 tokens is still less than a tile's whole row of blocks one after the other.
// Streamed / in tiles, k experts a token of E of 704 x 2816, gate and up: E = 128, k = 8: 64 tokens 59 / 95 us, 192 99 / 118,
// 256 119 / 122, 320 134 / 125; E = 32, k = 4 (256 tokens: 256 workgroups): 256 tokens 60 / 73, 400 82 / 70; E = 8, k = 2: 96
// tokens 28 / 47, 400 49 / 71 (past 100 tokens an expert: 500 52 / 74, 800 73 / 75; E = 2, k = 1: 300 27 / 69).  Down, E =
// 128, k = 8: 40 tokens 41 / 49, 96 58 / 58, 160 66 / 62; E = 8, k = 2: 32 22 / 18.
template <bool DOWN>
bool streams(const ExpertArgs &a)
{
    const int n = a.batch * a.k;
    if (a.cols / 32 > kStreamBlocks) return false;
    if (n <= (DOWN ? 6 : 16) * a.n_experts) return true;
    return !DOWN && n <= 100 * a.n_experts && (int64_t)max_tiles(a) * row_wgs<DOWN>(a) <= 256;  // n * cols < 2^27
}

template <bool DOWN>
int launch_stream(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    const int n = a.batch * a.k, nb = a.cols / 32, rows = 16 * kWaves * (DOWN ? stream_units<DOWN>() : 1);
    // the tokens of a tile: room for more costs workgroups on a CU, fewer of them passes over the weights.  8 / 16, 128
    // experts, eight a token, 20, 40, 64, 80, 96 tokens, in us: gate and up 36 / 41, 49 / 52, 57 / 60, 62 / 63, 70 / 67; down
    // 29.1 / 30.1, 39.8 / 37.9, 48.1 / 44.2, 52.2 / 48.0, 58.2 / 52.4.  Eight experts, two a token, 16, 20 tokens: gate and
    // up 20.1 / 20.3, 20.2 / 21.2; down 17.7 / 18.0, 17.9 / 19.0.
    const int tokens = n <= 4 * a.n_experts ? 8 : kStreamTokens;
    const dim3 grid((a.rows + rows - 1) / rows, std::min(n, n / tokens + a.n_experts));
#define MOE_STREAM(AT_ONCE, PART)                                                                            \
    hipLaunchKernelGGL((moe_stream_kernel<DOWN, AT_ONCE>), grid, dim3(64 * kWaves), stream_lds(nb, tokens, PART), \
                       ctx->stream, a, tokens)
    // Whole units / runs of 128 bytes a row, 40 tokens, 128 experts, eight a token: down of 2816 rows of 22 blocks 40 / 45 us,
    // of 30 54 / 58, of 24 (whole lines as it is) 42 / 41, of 32 48 / 48.  An expert's scales have to begin at 16 bytes.
    if (nb <= kWholeBlocks && nb % 8 && (int64_t)a.rows * nb % 8 == 0) MOE_STREAM(0, whole_part(nb));
    else if (nb % 8 == 0) MOE_STREAM(8, kBounce);
    else if (nb % 4 == 0) MOE_STREAM(4, kBounce);
    else if (nb % 2 == 0) MOE_STREAM(2, kBounce);
    else MOE_STREAM(1, kBounce);
#undef MOE_STREAM
    return check_launch(ctx, "moe_stream_kernel");
}

int launch_combine(mrml_hip_ctx *ctx, const ExpertArgs &a, float *y)
{
    if (a.rows % 4 == 0)
        hipLaunchKernelGGL(moe_combine_kernel<4>, dim3(a.batch, (a.rows / 4 + 255) / 256), dim3(256), 0, ctx->stream, a, y);
    else
        hipLaunchKernelGGL(moe_combine_kernel<1>, dim3(a.batch, (a.rows + 255) / 256), dim3(256), 0, ctx->stream, a, y);
    return check_launch(ctx, "moe_combine_kernel");
}

// The product itself: activations in MFMA order and the list of tiles in the workspace, then the tiles.
template <bool DOWN>
int launch_product(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    const int most = max_tiles(a), nb = a.cols / 32, n = a.batch * a.k, rows = DOWN ? n : a.batch;
    // a launch has less than 2^32 threads
    REQUIRE(ctx, tile_grid<DOWN>(a, most) * 64 * kWaves <= UINT32_MAX, "moe: batch * k = %d assignments of %d rows are too "
            "many for one call", n, a.rows);
    const size_t list = align_up((size_t)(1 + most) * sizeof(Tile), 256), scales = align_up((size_t)rows * 4, 256);
    const size_t packed = (size_t)rows * nb * kXBlock, part = DOWN ? align_up((size_t)n * a.rows * 4, 16) : 0;
    uint8_t *ws = (uint8_t *)workspace(ctx, list + scales + packed + part + (DOWN ? (size_t)n * 4 : 0));
    if (!ws) return MRML_HIP_E_ALLOC;
    Tile *tiles = (Tile *)ws;
    float *xscale = (float *)(ws + list);
    uint8_t *xp = ws + list + scales;
    // more than 1024 values: four waves a row, so that few long rows fill the chip as well (1501 rows of 2816: 12 us, one
    // wave a row 16)
    const int check_wgs = (n + 255) / 256, waves = a.cols <= 1024 ? 1 : 4;
    const dim3 grid(1 + check_wgs + (rows * waves + 3) / 4), block(256);
    ExpertArgs p = a;
    if (DOWN) p.named = (int32_t *)(xp + packed + part);
#define PACK(...)                                                                                             \
    hipLaunchKernelGGL((moe_pack_kernel<__VA_ARGS__>), grid, block, 0, ctx->stream, p, rows, check_wgs, xp, xscale, tiles)
    if (a.xpack && waves == 1) PACK(true, 1, 0);
    else if (a.xpack) PACK(true, 4, 0);
    else if (waves == 1) PACK(false, 1, 4);
    else if (a.cols <= 4096) PACK(false, 4, 4);
    else PACK(false, 4, 0);
#undef PACK
    if (int rc = check_launch(ctx, "moe_pack_kernel")) return rc;
    if (DOWN) p.out = (float *)(xp + packed);
    if (int rc = launch_tiles<DOWN>(ctx, p, most, tiles, xp, xscale)) return rc;
    return DOWN ? launch_combine(ctx, p, a.out) : MRML_HIP_OK;
}

}  // namespace

int launch_moe_gate_up(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    if (one_by_one(a)) return launch_gate_up_one(ctx, a);
    if (!streams<false>(a)) return launch_product<false>(ctx, a);
    ExpertArgs p = a;
    if (!p.xpack) {
        uint8_t *pack = (uint8_t *)workspace(ctx, act_pack_bytes((size_t)a.batch * (a.cols / 32)));
        if (!pack) return MRML_HIP_E_ALLOC;
        if (int rc = launch_quantize_q8_0(ctx, a.x, nullptr, pack, a.batch * a.cols)) return rc;
        p.xpack = pack;
    }
    return launch_stream<false>(ctx, p);
}

int launch_moe_down(mrml_hip_ctx *ctx, const ExpertArgs &a)
{
    if (one_by_one(a)) return launch_down_one(ctx, a);
    if (!streams<true>(a)) return launch_product<true>(ctx, a);
    const int n = a.batch * a.k;
    const size_t part = align_up((size_t)n * a.rows * 4, 16), pack = align_up(act_pack_bytes(n * (a.cols / 32)), 16);
    uint8_t *ws = (uint8_t *)workspace(ctx, part + pack + (size_t)n * 4);
    if (!ws) return MRML_HIP_E_ALLOC;
    if (int rc = launch_quantize_q8_0(ctx, a.x, nullptr, ws + part, n * a.cols)) return rc;
    ExpertArgs p = a;
    p.xpack = ws + part;
    p.out = (float *)ws;
    p.named = (int32_t *)(ws + part + pack);
    if (int rc = launch_stream<true>(ctx, p)) return rc;
    return launch_combine(ctx, p, a.out);
}

}  // namespace mrml
