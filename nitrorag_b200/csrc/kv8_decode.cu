// Decode attention over e4m3 pages (nr_paged_attention_decode_kv8).
//
// One query row per sequence: every cached byte is used once for each of the query heads
// that share it, so the kernel is bound by reading the pages.  A page's 16 tokens are the
// M = 16 rows of mma.m16n8k16 and up to 8 query heads of a group its N = 8 columns:
//
//   S^T[token][head] = K[token][dim] Q^T[dim][head]
//   O^T[dim][head]  += V^T[dim][token] W[token][head]
//
// e4m3 values are exact in fp16, so K and V enter the products unrounded (one conversion
// for two values).  The order of the summed dims and tokens is free, which lets each lane
// load 16 contiguous bytes of its rows straight from global memory into fragment order: no
// shared memory, and no barrier between the warps until the end.
//
// fp16 has few exponent bits, so both small operands are scaled by powers of two (exact):
// a query row to a largest value of 2^7, and the weights W = p * v_scale * gain with a gain
// per head that puts the largest weight so far near 2^7, whatever the blocks' scales are.
// Weights down to 2^-21 of the largest keep fp16's relative precision, smaller ones are off by
// at most 2^-32 of the largest (which shows only in a dim where the tokens with the large
// weights have no values).  p = exp2(s - m) goes by a
// running maximum that is only moved when a score passes it by 8 (a weight of at most 2^8
// costs no precision), so most pages need no exchange between lanes.  16-bit inputs round
// a weight once to fp16 (2^-11, under a bf16 output's own rounding and as much as an fp16
// one's); fp32 inputs carry query and weights as two fp16 halves (22 bits) and take each
// product twice.
//
// Work: the pages of all (sequence, kv head) items are cut into units of about equal
// length, one CTA each, its four warps taking every fourth page.  The cut goes by the
// lengths on the device, so a ragged batch and a table much wider than its contexts cost
// nothing.  An item of one unit is finished by its CTA.  The units of a longer one leave their
// maximum, sum and output in the workspace, joined in order (the result does not depend on
// who finishes last): up to kJoinItems items, each of many parts, by a second kernel with a
// CTA for each head (2 sequences of 57k tokens, 16 heads on one: 87 -> 23 us; 4096 tokens, 8
// items: 13.5 -> 10.2; but at 64 items 26.5 -> 27.0); else by the item's last CTA.
//
// Measured (of the copy bandwidth): 2 contexts of 131k tokens, 32 heads on 8, head_dim 128,
// fp16: 104 us, 5.2 TB/s (0.79; issue slots are 40 % busy, mostly converting the codes).  96
// contexts of 0..4096 tokens, the same heads: 101 us, 4.2 TB/s (0.64): a page's scales and
// codes are addressed by a table entry that has to be read first, and a unit's start and end
// read nothing.  64 contexts of 128..1024, 12 heads of 64, fp32: 25 us, 2.3 TB/s (0.35): each
// item is one unit, and a warp of the longest takes its 16 pages one after another.  One
// context of 601 tokens: 8 us, a unit's chain of latencies.
// Tried and left: runs of equal length over item borders, several items' pieces to a CTA
// (27 -> 36, 100 -> 115 us: the pieces' latencies come one after another).
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"

namespace nitro {

namespace {

constexpr int kWarps = 4;
constexpr int kWaves = 2;
constexpr int kSms = 148, kMostCtas = 5;
// Pages are cut into so many units, `slots` of which run at once.  With few items the last
// units should not start a second wave (each item can add one unit to the even cut); many
// items run in several waves anyway, which smaller units even out.
__host__ __device__ __forceinline__ int units_wanted(int64_t items, int slots) {
    return items <= slots / 2 ? slots - (int)items : kWaves * slots;
}
// A unit's least pages: two for each warp where items are few, more where items alone fill the
// device.  With 8 and with 64 pages at least, 8 kv heads of 128, bf16, 1000 tokens: 16 / 18
// sequences 14.5 / 16.4 us with 8 (what the rule takes); 19 / 24 / 32: 16.5 / 17.1 / 20.6
// with 8, 23.5 / 24.5 / 26.3 with 64 (taken); 48 / 64: 32.7 / 43.6 with 8, 30.1 / 30.9 with 64
// (taken).  12 heads of 64, fp32, 128..1024 tokens: 24 sequences 14.6 and 20.6 (taken), 32:
// 23.7 and 22.1 (taken), 64: 31.3 and 24.7 (taken).  So from 149 to about 300 items, half the
// CTAs that run at once, the rule takes the slower side.
constexpr int kMinPages = 8, kMinPagesMany = 64;
__host__ __device__ __forceinline__ int least_pages(int64_t items) { return items <= kSms ? kMinPages : kMinPagesMany; }
// Items whose partial results can be counted; more items than that fill the device uncut.
constexpr int kCounters = 16384;
constexpr int kJoinItems = 32;  // most items whose parts a second kernel joins
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two e4m3 codes (low and high byte) as fp16, exact.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint16_t c) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(c));
    return d;
}
__device__ __forceinline__ void word_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = e4m3x2_f16x2((uint16_t)w);
    hi = e4m3x2_f16x2((uint16_t)(w >> 16));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// What is left of two values after their rounding to fp16 in h.
__device__ __forceinline__ uint32_t pack_f16_rest(float lo, float hi, uint32_t h) {
    const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return pack_f16(lo - r.x, hi - r.y);
}

__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8x8 matrix of 16-bit values held one row to four lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

__device__ __forceinline__ uint4 load16(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load8(const uint8_t* p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// 2^(7 - exponent of x), within the normal range; 1 for zero, infinities and NaN.
__device__ __forceinline__ float gain_of(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 0xff);
    if (!(x > 0.0f) || e == 255) return 1.0f;
    return __uint_as_float((uint32_t)min(max(261 - e, 2), 252) << 23);
}

// A lane's part of a page of K and of V: with g = lane / 4, c = lane % 4, bytes 16c.. of each
// 64 of K's rows g and g + 8, and bytes g*HD/8.. of V's rows 2c, 2c+1, 2c+8, 2c+9.
template <int HD>
struct KeyRegs {
    uint32_t w[2][HD / 64][4];
    __device__ __forceinline__ void load(const uint8_t* tile, int g, int c) {
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int j = 0; j < HD / 64; j++) {
                const uint4 u = load16(tile + (g + 8 * r) * HD + 64 * j + 16 * c);
                w[r][j][0] = u.x; w[r][j][1] = u.y; w[r][j][2] = u.z; w[r][j][3] = u.w;
            }
    }
};
template <int HD>
struct ValueRegs {
    uint32_t w[4][HD / 32];
    __device__ __forceinline__ void load(const uint8_t* tile, int g, int c) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint8_t* p = tile + (2 * c + (t & 1) + 8 * (t >> 1)) * HD + g * (HD / 8);
            if constexpr (HD == 128) {
                const uint4 u = load16(p);
                w[t][0] = u.x; w[t][1] = u.y; w[t][2] = u.z; w[t][3] = u.w;
            } else {
                const uint2 u = load8(p);
                w[t][0] = u.x; w[t][1] = u.y;
            }
        }
    }
};

// Running state of one warp: NT tiles of 8 heads; a lane's columns are heads 2c, 2c + 1 of
// each, its output rows dims g*HD/8 .. + HD/8 - 1.
template <int HD, int NT, bool SPLIT>
struct WarpState {
    uint32_t q[SPLIT ? 2 : 1][NT][HD / 64][8];
    float o[NT][HD / 16][4];
    float m[NT][2], l[NT][2], wmax[NT][2], gain[NT][2], factor[NT][2];

    // Scores of one page; two sums side by side halve the chain of products.
    __device__ __forceinline__ void scores(const KeyRegs<HD>& k, float (&s)[NT][4]) {
        float s2[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[n][i] = s2[n][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                uint32_t a0, a1, a2, a3;
                word_f16(k.w[0][j][w], a0, a2);
                word_f16(k.w[1][j][w], a1, a3);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    mma_f16((w & 1) && !SPLIT ? s2[n] : s[n], a0, a1, a2, a3, q[0][n][j][2 * w], q[0][n][j][2 * w + 1]);
                    if constexpr (SPLIT) mma_f16(s2[n], a0, a1, a2, a3, q[1][n][j][2 * w], q[1][n][j][2 * w + 1]);
                }
            }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[n][i] += s2[n][i];
    }

    // Scores to weights, as the second product's operand.
    __device__ __forceinline__ void weights(float (&s)[NT][4], float ks, float vs, int valid, int g,
                                            uint32_t (&b)[SPLIT ? 2 : 1][NT][2]) {
        bool moves = false;
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int i = 0; i < 4; i++) s[n][i] *= ks * factor[n][i & 1];
            if (valid < kPage) {
                if (g >= valid) s[n][0] = s[n][1] = -INFINITY;
                if (g + 8 >= valid) s[n][2] = s[n][3] = -INFINITY;
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
                moves |= fmaxf(s[n][h], s[n][2 + h]) > m[n][h] + 8.0f || vs * gain[n][h] > 128.0f;
        }
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float t = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
                    const float mn = fmaxf(m[n][h], t);
                    const float corr = m[n][h] == -INFINITY ? 0.0f : exp2_fast(m[n][h] - mn);
                    const float now = t == -INFINITY ? 0.0f : exp2_fast(t - mn) * vs;
                    wmax[n][h] = fmaxf(wmax[n][h] * corr, now);
                    const float next = gain_of(wmax[n][h]);
                    const float f = corr * next * (1.0f / gain[n][h]);
                    l[n][h] *= corr;
#pragma unroll
                    for (int i = 0; i < HD / 16; i++) {
                        o[n][i][h] *= f;
                        o[n][i][2 + h] *= f;
                    }
                    m[n][h] = mn;
                    gain[n][h] = next;
                }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = exp2_fast(s[n][i] - m[n][i & 1]);
                l[n][i & 1] += p;
                w[i] = p * vs * gain[n][i & 1];  // vs * gain alone may pass the range: a scale of 2^-126 so far
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t hi = pack_f16(w[2 * i], w[2 * i + 1]);
                b[0][n][i] = transpose8(hi);
                if constexpr (SPLIT) b[1][n][i] = transpose8(pack_f16_rest(w[2 * i], w[2 * i + 1], hi));
            }
        }
    }

    __device__ __forceinline__ void add_values(const ValueRegs<HD>& r, const uint32_t (&b)[SPLIT ? 2 : 1][NT][2], int valid, int c) {
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
            // bytes 2i, 2i + 1 of the lane's 4 rows: adjacent tokens' values of a dim side by side
            const uint32_t sel = (i & 1) ? 0x7362 : 0x5140;
            uint32_t v0 = r.w[0][i / 2], v1 = r.w[1][i / 2], v2 = r.w[2][i / 2], v3 = r.w[3][i / 2];
            if (valid < kPage) {  // what lies behind the last token may be NaN
                if (2 * c >= valid) v0 = 0;
                if (2 * c + 1 >= valid) v1 = 0;
                if (2 * c + 8 >= valid) v2 = 0;
                if (2 * c + 9 >= valid) v3 = 0;
            }
            uint32_t a0, a1, a2, a3;
            word_f16(__byte_perm(v0, v1, sel), a0, a1);
            word_f16(__byte_perm(v2, v3, sel), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                mma_f16(o[n][i], a0, a1, a2, a3, b[0][n][0], b[0][n][1]);
                if constexpr (SPLIT) mma_f16(o[n][i], a0, a1, a2, a3, b[1][n][0], b[1][n][1]);
            }
        }
    }
};

__device__ __forceinline__ int context_of(const Kv8DecodeArgs& a, int b, bool& bad) {
    const int64_t n = a.ctx_lens[b], cap = (int64_t)a.max_pages * kPage;
    bad = n < 0 || n > cap;
    return (int)(((n < 0 ? 0 : n > cap ? cap : n) + kPage - 1) / kPage);
}

// exp2(m - top), for a part without tokens 0 (or its NaN).
__device__ __forceinline__ float part_weight(float m, float top, float l) {
    return m == -INFINITY ? (l != l ? l : 0.0f) : exp2_fast(m - top);
}

// CTAs on an SM, by the registers a warp's state takes.
template <typename T, int HD, int NT>
constexpr int kCtas = NT == 2 ? (HD == 128 ? 2 : 3) : HD == 64 ? 5 : sizeof(T) == 4 ? 3 : 4;

// Floats of a unit's partial result: group rows of HD values, then the group's maxima and
// sums, a whole number of 16-byte pieces.
__host__ __device__ __forceinline__ int64_t partial_floats(int group, int head_dim) {
    return (int64_t)group * head_dim + (2 * group + 3) / 4 * 4;
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32, kCtas<T, HD, NT>) kv8_decode_kernel(Kv8DecodeArgs a, float* partial, int* counters, int2* items_cut) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int HEADS = 8 * NT, LD = HD + 4;
    __shared__ __align__(16) float s_o[kWarps][HEADS][LD], s_m[kWarps][HEADS], s_l[kWarps][HEADS];
    __shared__ int s_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int nkv = a.pool.n_kv_heads, group = a.n_heads / nkv;
    grid_dependency_wait();
    grid_dependents_launch();

    // the cut: all pages over the units wanted, then the sequence this unit belongs to
    int64_t total = 0;
    bool any_bad = false;
    int first_n = 0;  // pages of sequence `lane`
    for (int i = lane; i < a.B; i += 32) {
        bool bad;
        const int n = context_of(a, i, bad);
        if (i == lane) first_n = n;
        total += n;
        any_bad |= bad;
    }
    if (a.B <= 32) {  // at most 2^31 together: one number to a lane
        total = __reduce_add_sync(0xffffffffu, (uint32_t)total);
    } else {
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    }
    if (blockIdx.x == 0 && any_bad) flag_error(a.err, kErrBadContext);
    const int64_t items = (int64_t)a.B * nkv;
    const int wanted = units_wanted(items, kSms * kCtas<T, HD, NT>);
    const int64_t all = total * nkv;
    const int per = all <= INT32_MAX - wanted ? ((int)all + wanted - 1) / wanted : (int)min((all + wanted - 1) / wanted, (int64_t)INT32_MAX);
    const int chunk = items > kCounters ? INT32_MAX : max(least_pages(items), per);
    const int unit = blockIdx.x;
    int b = -1, pages = 0, units = 0, at = 0;  // at: first unit of sequence b
    for (int i0 = 0, before = 0; i0 < a.B && b < 0; i0 += 32) {
        const int i = i0 + lane;
        bool bad;
        const int n = i0 == 0 ? first_n : i < a.B ? context_of(a, i, bad) : 0;
        const int u = i < a.B ? max(0, n - 1) / chunk + 1 : 0;  // an empty row is written too
        int sum = u;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, x);
            if (lane >= x) sum += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, (int64_t)(before + sum) * nkv > unit);
        if (past) {
            const int src = __ffs(past) - 1;
            b = i0 + src;
            pages = __shfl_sync(0xffffffffu, n, src);
            units = __shfl_sync(0xffffffffu, u, src);
            at = before + __shfl_sync(0xffffffffu, sum - u, src);
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (b < 0) return;
    const int kvh = (unit - at * nkv) % nkv, part = (unit - at * nkv) / nkv;
    const int each = (pages + units - 1) / units;
    const int pg0 = part * each, pg1 = min(pages, pg0 + each);
    const int ctx = min(max(a.ctx_lens[b], 0), pages * kPage);

    // this warp's pages, 32 at a time: lane i looks up the i-th one's block and scales
    const int mine = pg1 - pg0 > warp ? (pg1 - pg0 - warp + kWarps - 1) / kWarps : 0;
    struct Lookup {
        int64_t block;
        float ks, vs;
    };
    auto look_up = [&](int base) {
        Lookup x{-1, 0.0f, 0.0f};
        if (base + lane < mine) {
            const int pg = pg0 + warp + kWarps * (base + lane);
            const int id = a.block_tables[(int64_t)b * a.max_pages + pg];
            if (id >= 0 && id < a.pool.n_pages) {
                x.block = ((int64_t)id * a.pool.n_layers + a.layer) * nkv + kvh;
                x.ks = a.pool.k_scale[x.block];
                x.vs = a.pool.v_scale[x.block];
            } else {
                flag_error(a.err, kErrBadContext);
            }
        }
        return x;
    };
    Lookup now = look_up(0), next{-1, 0.0f, 0.0f};
    KeyRegs<HD> kr;
    ValueRegs<HD> vr;
    int64_t block = __shfl_sync(0xffffffffu, now.block, 0);
    if (block >= 0) {
        kr.load(a.pool.k + block * (kPage * HD), g, c);
        vr.load(a.pool.v + block * (kPage * HD), g, c);
    }

    // the queries, while the first page is on its way
    WarpState<HD, NT, SPLIT> st;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int head = 8 * n + g;
        float x[HD / 64][16], top = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
            if (head < group) {
                const T* p = (const T*)a.q + ((int64_t)b * a.n_heads + kvh * group + head) * HD + 64 * j + 16 * c;
#pragma unroll
                for (int v = 0; v < (int)sizeof(T); v++) {
                    const uint4 u = reinterpret_cast<const uint4*>(p)[v];
                    const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
                    for (int i = 0; i < 16 / (int)sizeof(T); i++) x[j][v * (16 / (int)sizeof(T)) + i] = to_f32(t[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) x[j][i] = 0.0f;
            }
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, fabsf(x[j][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float up = std::is_same<T, __half>::value ? 1.0f : gain_of(top);
#pragma unroll
        for (int j = 0; j < HD / 64; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x0 = x[j][2 * i] * up, x1 = x[j][2 * i + 1] * up;
                st.q[0][n][j][i] = pack_f16(x0, x1);
                if constexpr (SPLIT) st.q[1][n][j][i] = pack_f16_rest(x0, x1, st.q[0][n][j][i]);
            }
        const float down = (1.0f / up) * (kLog2e * rsqrtf((float)HD));
#pragma unroll
        for (int h = 0; h < 2; h++) {
            st.factor[n][h] = __shfl_sync(0xffffffffu, down, (2 * c + h) * 4);
            st.m[n][h] = -INFINITY;
            st.l[n][h] = st.wmax[n][h] = 0.0f;
            st.gain[n][h] = 1.0f;
        }
#pragma unroll
        for (int i = 0; i < HD / 16; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) st.o[n][i][k] = 0.0f;
    }

    // A page's keys are replaced by the next page's as soon as they are used, its values too.
    for (int i = 0; i < mine; i++) {
        if (i % 32 == 0) next = look_up(i + 32);
        const float ks = __shfl_sync(0xffffffffu, now.ks, i % 32), vs = __shfl_sync(0xffffffffu, now.vs, i % 32);
        if (i % 32 == 31) now = next;
        const int64_t following = __shfl_sync(0xffffffffu, now.block, (i + 1) % 32);  // -1 behind the last
        const int left = ctx - (pg0 + warp + kWarps * i) * kPage;
        float s[NT][4];
        uint32_t w[SPLIT ? 2 : 1][NT][2];
        if (block >= 0) st.scores(kr, s);
        if (following >= 0) kr.load(a.pool.k + following * (kPage * HD), g, c);
        if (block >= 0) {
            st.weights(s, ks, vs, left, g, w);
            st.add_values(vr, w, left, c);
        }
        if (following >= 0) vr.load(a.pool.v + following * (kPage * HD), g, c);
        block = following;
    }

    // join the warps
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float l = st.l[n][h];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            const int head = 8 * n + 2 * c + h;
            if (g == 0) s_m[warp][head] = st.m[n][h], s_l[warp][head] = l;
            const float down = 1.0f / st.gain[n][h];
#pragma unroll
            for (int i = 0; i < HD / 16; i++) {
                float2 v = make_float2(st.o[n][i][h] * down, st.o[n][i][2 + h] * down);
                *reinterpret_cast<float2*>(&s_o[warp][head][g * (HD / 8) + 2 * i]) = v;
            }
        }
    __syncthreads();
    const int64_t rec = partial_floats(group, HD);
    float* mine_out = partial + (int64_t)unit * rec;
    T* out = (T*)a.out + ((int64_t)b * a.n_heads + kvh * group) * HD;
    for (int e = threadIdx.x * 4; e < group * HD; e += blockDim.x * 4) {
        const int head = e / HD, d = e % HD;
        float top = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWarps; w++) top = fmaxf(top, s_m[w][head]);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = part_weight(s_m[w][head], top, s_l[w][head]);
            l += f * s_l[w][head];
            const float4 v = *reinterpret_cast<const float4*>(&s_o[w][head][d]);
            acc[0] += f * v.x; acc[1] += f * v.y; acc[2] += f * v.z; acc[3] += f * v.w;
        }
        if (units == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int i = 0; i < 4; i++) out[e + i] = from_f32<T>(acc[i] * inv);
        } else {
            *reinterpret_cast<float4*>(mine_out + e) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (d == 0) mine_out[group * HD + head] = top, mine_out[group * HD + group + head] = l;
        }
    }
    if (items_cut) {
        if (part == 0 && threadIdx.x == 0) items_cut[b * nkv + kvh] = make_int2(unit, units);
        return;
    }
    if (units == 1) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        // release: what the CTA wrote before the barrier; acquire: what the others did
        int* n = counters + b * nkv + kvh;
        int before;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(n) : "memory");
        s_last = before == units - 1;
        if (s_last) *n = 0;
    }
    __syncthreads();
    if (!s_last) return;
    // the weights of the parts: a warp for each head, a lane for each part
    const float* first = partial + ((int64_t)at * nkv + kvh) * rec;
    const int64_t step = (int64_t)nkv * rec;
    for (int head = warp; head < group; head += kWarps) {
        float top = -INFINITY;
        for (int u = lane; u < units; u += 32) top = fmaxf(top, __ldcg(first + u * step + group * HD + head));
        top = warp_max(top);
        float l = 0.0f;
        for (int u = lane; u < units; u += 32) {
            const float pl = __ldcg(first + u * step + group * HD + group + head);
            l += part_weight(__ldcg(first + u * step + group * HD + head), top, pl) * pl;
        }
        l = warp_sum(l);
        if (lane == 0) s_m[0][head] = top, s_l[0][head] = l == 0.0f ? 0.0f : 1.0f / l;
    }
    __syncthreads();
    for (int e = threadIdx.x * 4; e < group * HD; e += blockDim.x * 4) {
        const int head = e / HD;
        const float top = s_m[0][head], inv = s_l[0][head];
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int u0 = 0; u0 < units; u0 += 8) {
            float4 v[8];
            float m[8], l[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float* p = first + min(u0 + i, units - 1) * step;
                v[i] = __ldcg(reinterpret_cast<const float4*>(p + e));
                m[i] = __ldcg(p + group * HD + head);
                l[i] = __ldcg(p + group * HD + group + head);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // a weight of 0 too: a NaN reaches the row whatever its weight
                const float f = u0 + i < units ? part_weight(m[i], top, l[i]) : 0.0f;
                if (u0 + i < units) {
                    acc[0] += f * v[i].x; acc[1] += f * v[i].y; acc[2] += f * v[i].z; acc[3] += f * v[i].w;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) out[e + i] = from_f32<T>(acc[i] * inv);
    }
}

// The parts of one head's item: `items_cut` has an item's first unit and how many it has.
template <typename T, int HD>
__global__ void __launch_bounds__(128) kv8_join_kernel(Kv8DecodeArgs a, const float* partial, const int2* items_cut) {
    constexpr int LANES = HD / 4, SLICES = 128 / LANES;  // four dims to a thread, every SLICES-th part
    __shared__ __align__(16) float s_o[SLICES][HD];
    __shared__ float s_l[SLICES], s_top;
    const int nkv = a.pool.n_kv_heads, group = a.n_heads / nkv;
    const int b = blockIdx.x / a.n_heads, head = blockIdx.x % a.n_heads, kvh = head / group, in_group = head % group;
    const int lane = threadIdx.x % LANES, slice = threadIdx.x / LANES;
    grid_dependency_wait();
    grid_dependents_launch();
    const int2 cut = items_cut[b * nkv + kvh];
    const int units = cut.y;
    if (units <= 1) return;
    const int64_t rec = partial_floats(group, HD), step = nkv * rec;
    const float* first = partial + cut.x * rec;
    const float* m_of = first + group * HD + in_group;
    if (threadIdx.x < 32) {
        float top = -INFINITY;
        for (int u = threadIdx.x; u < units; u += 32) top = fmaxf(top, m_of[u * step]);
        top = warp_max(top);
        if (threadIdx.x == 0) s_top = top;
    }
    __syncthreads();
    const float top = s_top;
    float l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int u = slice; u < units; u += SLICES) {
        const float4 v = *reinterpret_cast<const float4*>(first + u * step + in_group * HD + 4 * lane);
        const float pl = m_of[u * step + group], f = part_weight(m_of[u * step], top, pl);
        l += f * pl;
        acc[0] += f * v.x; acc[1] += f * v.y; acc[2] += f * v.z; acc[3] += f * v.w;
    }
    *reinterpret_cast<float4*>(&s_o[slice][4 * lane]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (lane == 0) s_l[slice] = l;
    __syncthreads();
    if (threadIdx.x < HD) {
        float sum = 0.0f, o = 0.0f;
#pragma unroll
        for (int i = 0; i < SLICES; i++) sum += s_l[i], o += s_o[i][threadIdx.x];
        ((T*)a.out)[((int64_t)b * a.n_heads + head) * HD + threadIdx.x] = from_f32<T>(sum == 0.0f ? 0.0f : o / sum);
    }
}

template <typename T, int HD, int NT>
cudaError_t launch_nt(const Kv8DecodeArgs& a, cudaStream_t s) {
    int* counters = (int*)a.workspace;
    float* partial = (float*)((char*)a.workspace + kCounters * sizeof(int));
    const int64_t items = (int64_t)a.B * a.pool.n_kv_heads;
    // No more CTAs than the table has room for units: an idle one takes the time of its look at
    // the lengths.
    const int64_t most = items > kCounters ? items : items * ((a.max_pages - 1) / least_pages(items) + 1);
    const dim3 grid((unsigned)std::min(items + units_wanted(items, kSms * kCtas<T, HD, NT>), most));
    // Up to 8 parts are loaded at once by the last CTA: not worth a second launch (601 tokens, 12
    // items: 8.7 us a call, 10.1 with it).
    const bool join = items <= kJoinItems && a.max_pages > 8 * kMinPages;
    int2* items_cut = join ? (int2*)(partial + (items + kWaves * kSms * kMostCtas) * partial_floats(a.n_heads / a.pool.n_kv_heads, HD)) : nullptr;
    const cudaError_t rc = launch_ex(kv8_decode_kernel<T, HD, NT>, grid, dim3(kWarps * 32), 0, s, 1, a, partial, counters, items_cut);
    if (rc != cudaSuccess || !join) return rc;
    count_launch();
    return launch_ex(kv8_join_kernel<T, HD>, dim3((unsigned)a.B * a.n_heads), dim3(128), 0, s, 1, a, (const float*)partial, (const int2*)items_cut);
}

template <typename T, int HD>
cudaError_t launch_hd(const Kv8DecodeArgs& a, cudaStream_t s) {
    return a.n_heads / a.pool.n_kv_heads <= 8 ? launch_nt<T, HD, 1>(a, s) : launch_nt<T, HD, 2>(a, s);
}

template <typename T>
cudaError_t launch_t(const Kv8DecodeArgs& a, cudaStream_t s) {
    return a.pool.head_dim == 64 ? launch_hd<T, 64>(a, s) : launch_hd<T, 128>(a, s);
}

}  // namespace

size_t kv8_decode_workspace_bytes(int B, int n_heads, int n_kv_heads, int head_dim, int) {
    const size_t rec = partial_floats(n_heads / n_kv_heads, head_dim) * sizeof(float);
    // the largest cut batch up to B: what holds a batch holds every smaller one, also where B's own
    // items are past the counters and need no partial results
    const int64_t items = std::min(B, kCounters / n_kv_heads) * (int64_t)n_kv_heads;
    const size_t n = items ? (size_t)(items + kWaves * kSms * kMostCtas) * rec : 0;
    return kCounters * sizeof(int) + (n + 255) / 256 * 256 + kJoinItems * sizeof(int2);
}

cudaError_t launch_kv8_decode(const Kv8DecodeArgs& a, cudaStream_t s) {
    count_launch();
    if (a.dtype == kF32) return launch_t<float>(a, s);
    if (a.dtype == kBF16) return launch_t<__nv_bfloat16>(a, s);
    return launch_t<__half>(a, s);
}

}  // namespace nitro
