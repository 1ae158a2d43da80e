// Append of rotated keys and values to e4m3 pages (nr_kv8_append).
//
// A CTA takes a unit, the part of one page that a sequence's new tokens fall into (at most 16
// tokens), and some or all of its heads: of q, k and v, one head's 16 x head_dim tile to a
// warp at a time, held in registers in the input's type.  One read of the input serves the
// rotation, the outputs, the block's maximum and, turned once more, the codes.  The unit's
// sines and cosines wait in shared memory for all heads, and a warp's next tile is on its way
// while it works on one.
//
// Scale of a block: the smallest 2^e with |x| <= 448 * 2^e (448 is the largest e4m3 value).
// With |x|max = 1.m * 2^E and 448 = 1.75 * 2^8 that is e = E - 8, one more if 1.m > 1.75:
// read off the float's bits.  e4m3 keeps its relative precision over 2^14, so rounding the
// scale up to a power of two loses no accuracy, and dividing by it is exact: a block that
// grows token by token ends with the codes it would have got at once (but for values that
// fall below the normal range), and the older codes are not rounded again and again.
// The maximum is taken over the bits of |x| as unsigned numbers, in which infinities and
// NaNs are largest: they reach the scale, which becomes NaN.
//
// Measured: 12 prompts of 33..1300 tokens (8k together), 32 heads on 8 of 128, bf16: 49 us,
// 5.0 TB/s, 0.76 of the measured copy bandwidth; reads and writes alternate in each warp,
// and issue slots are a third to half busy with the rotation and the conversions.  One token
// of 61 sequences: 7.4 us, of one: 3.6 us, the chain from the lengths over the page table to
// the page (a call costs the host 8 us).  A CTA for each unit and head, the tile in fp32: 80 us
// (a lane's 64 values leave registers for few warps).
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"

namespace nitro {

namespace {

constexpr int kWarps = 4, kCtas = 5;  // warps of a CTA, CTAs on an SM
constexpr int kFill = 16;             // CTAs for each SM that a unit's heads are spread over

__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    const int biased = (int)(amax_bits >> 23);
    if (biased == 255) return __uint_as_float(0x7fc00000u);
    const int e = biased - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// Two fp32 values as e4m3 codes (round to nearest even), the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// 16 codes times r, as codes.
__device__ __forceinline__ uint4 recode(uint4 c, float r) {
    uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] & 0xffff), __NV_E4M3)));
        const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> 16), __NV_E4M3)));
        w[i] = e4m3x2(a.x * r, a.y * r) | (e4m3x2(b.x * r, b.y * r) << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
struct Vec {  // 16 bytes of input elements
    static constexpr int N = 16 / (int)sizeof(T);
    static __device__ __forceinline__ void unpack(const uint4& u, float* v) {
        const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = to_f32(t[i]);
    }
    static __device__ __forceinline__ void store(T* p, const float* v) {
        uint4 u;
        T* t = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = from_f32<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = u;
    }
    static __device__ __forceinline__ void store_codes(uint8_t* p, const float* v, float inv) {
        uint32_t w[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; i++)
            w[i] = e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) | (e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16);
        if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(p) = w[0];
    }
};

// What is turned: nothing, neighbours (2i, 2i + 1), or (i, i + rot_dim / 2).
enum Rot { kNone, kNeighbours, kHalves };

// Two vectors of a row, at elements e0 and e1, turned: two products and a sum for each element,
// each rounded.  cos, sin: the row's, rot_dim / 2 of them.
template <Rot ROT, int N>
__device__ __forceinline__ void rotate(float* x, float* y, const float* cos, const float* sin, int e0, int e1) {
    if constexpr (ROT == kHalves) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 c4 = *reinterpret_cast<const float4*>(cos + e0 + i), s4 = *reinterpret_cast<const float4*>(sin + e0 + i);
            const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float a = x[i + k], b = y[i + k];
                x[i + k] = __fsub_rn(__fmul_rn(a, cc[k]), __fmul_rn(b, ss[k]));
                y[i + k] = __fadd_rn(__fmul_rn(a, ss[k]), __fmul_rn(b, cc[k]));
            }
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float* v = h ? y : x;
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const int at = ((h ? e1 : e0) + i) / 2;
                const float2 c = *reinterpret_cast<const float2*>(cos + at), s = *reinterpret_cast<const float2*>(sin + at);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float cc = k ? c.y : c.x, ss = k ? s.y : s.x, a = v[i + 2 * k], b = v[i + 2 * k + 1];
                    v[i + 2 * k] = __fsub_rn(__fmul_rn(a, cc), __fmul_rn(b, ss));
                    v[i + 2 * k + 1] = __fadd_rn(__fmul_rn(a, ss), __fmul_rn(b, cc));
                }
            }
        }
    }
}

// The larger of m and |x|, NaN if x is.
__device__ __forceinline__ float max_abs(float m, float x) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(m), "f"(fabsf(x)));
    return d;
}

// The part of a page a CTA works on, and a lane's place in its rows: the vectors of a row are
// taken in pairs so that a lane holds both elements of every rotation pair, (j, j + half the
// rotated vectors) in the rotated part and the same split of the rest.
struct Unit {
    int64_t first;  // row of its first token
    int n, slot0;   // tokens, and rows of the page that are there already
    int r0, e0, e1; // first row, elements of the two vectors
    bool rotated;
};

template <typename T, int HD>
struct Tile {
    static constexpr int VE = Vec<T>::N;
    static constexpr int PAIRS = HD / (2 * VE);  // vector pairs in a row
    static constexpr int ROWS = 32 / PAIRS;      // rows a warp covers at a time
    static constexpr int STEPS = kPage / ROWS;
    uint4 v[STEPS][2];

    // Keeps the compiler from holding what it derived from the tile so far for its next use: the
    // 64 values of a lane would leave no registers for other warps.
    __device__ __forceinline__ void forget_derived() {
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int h = 0; h < 2; h++) asm volatile("" : "+r"(v[s][h].x), "+r"(v[s][h].y), "+r"(v[s][h].z), "+r"(v[s][h].w));
    }

    // Rows behind the last token repeat it: they change no maximum and are not stored.
    __device__ __forceinline__ void load(const T* src, int64_t ld, const Unit& u) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const T* row = src + (u.first + min(s * ROWS + u.r0, u.n - 1)) * ld;
            v[s][0] = *reinterpret_cast<const uint4*>(row + u.e0);
            v[s][1] = *reinterpret_cast<const uint4*>(row + u.e1);
        }
    }

    // Rotated (ROT) rows to dst (if there is one) and, with MAX, their largest |value|.
    template <Rot ROT, bool MAX>
    __device__ __forceinline__ float turn(T* dst, int64_t ld, const Unit& u, const float (*cos)[HD / 2], const float (*sin)[HD / 2]) const {
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int r = s * ROWS + u.r0;
            float x[VE], y[VE];
            Vec<T>::unpack(v[s][0], x);
            Vec<T>::unpack(v[s][1], y);
            if (ROT != kNone && u.rotated) rotate<ROT, VE>(x, y, cos[min(r, u.n - 1)], sin[min(r, u.n - 1)], u.e0, u.e1);
            if (dst && r < u.n) {
                T* row = dst + (u.first + r) * ld;
                Vec<T>::store(row + u.e0, x);
                Vec<T>::store(row + u.e1, y);
            }
            if (MAX) {
#pragma unroll
                for (int i = 0; i < VE; i++) top = max_abs(max_abs(top, x[i]), y[i]);
            }
        }
        return top;
    }

    // The block's codes, its older rows coded anew if its scale grows.
    template <Rot ROT>
    __device__ __forceinline__ void append(float top, float before, float* scale_at, uint8_t* codes, const Unit& u, const float (*cos)[HD / 2],
                                           const float (*sin)[HD / 2]) const {
        const int lane = threadIdx.x & 31;
        float scale = block_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu));
        if (u.slot0) {
            const bool grows = __float_as_uint(scale) > __float_as_uint(before);
            if (grows) {
                const float r = before / scale;
                for (int i = lane * 16; i < u.slot0 * HD; i += 32 * 16) {
                    uint4* c = reinterpret_cast<uint4*>(codes + i);
                    *c = recode(*c, r);
                }
            } else {
                scale = before;
            }
            if (grows && lane == 0) *scale_at = scale;
        } else if (lane == 0) {
            *scale_at = scale;
        }
        const float inv = 1.0f / scale;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int r = s * ROWS + u.r0;
            float x[VE], y[VE];
            Vec<T>::unpack(v[s][0], x);
            Vec<T>::unpack(v[s][1], y);
            if (ROT != kNone && u.rotated) rotate<ROT, VE>(x, y, cos[min(r, u.n - 1)], sin[min(r, u.n - 1)], u.e0, u.e1);
            if (r < u.n) {
                uint8_t* row = codes + (u.slot0 + r) * HD;
                Vec<T>::store_codes(row + u.e0, x, inv);
                Vec<T>::store_codes(row + u.e1, y, inv);
            }
        }
    }
};

template <typename T, int HD, Rot ROT>
__global__ void __launch_bounds__(kWarps * 32, kCtas) kv8_append_kernel(Kv8AppendArgs a) {
    using Tl = Tile<T, HD>;
    __shared__ __align__(16) float s_cos[kPage][HD / 2], s_sin[kPage][HD / 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    grid_dependents_launch();
    auto in_range = [&](int r0, int r1, int at) {
        const int64_t end = (int64_t)at + r1 - r0;
        return r0 >= 0 && r1 >= r0 && r1 <= a.T && at >= 0 && end <= (int64_t)a.max_pages * kPage && (ROT == kNone || end <= a.rope_len);
    };
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < a.B; i += blockDim.x)
            if (a.cu_seqlens[i] != a.cu_seqlens[i + 1] && !in_range(a.cu_seqlens[i], a.cu_seqlens[i + 1], a.start_pos[i]))
                flag_error(a.err, kErrBadContext);
    const int b = seq_of_unit<kPage, 2>(a.cu_seqlens, a.B, blockIdx.x, lane);
    const int row0 = a.cu_seqlens[b], row1 = a.cu_seqlens[b + 1], start = a.start_pos[b];
    const int j = (int)blockIdx.x - (row0 / kPage + 2 * b);
    if (j < 0 || row1 == row0) return;
    const int64_t end = (int64_t)start + row1 - row0;
    if (!in_range(row0, row1, start)) return;
    const int pg = start / kPage + j;
    if ((int64_t)pg * kPage >= end) return;
    const int pos0 = max(start, pg * kPage);
    const int rot_pairs = a.rot_dim / (2 * Tl::VE), p = lane % Tl::PAIRS;
    Unit u;
    u.n = (int)min(end, (int64_t)(pg + 1) * kPage) - pos0;
    u.slot0 = pos0 - pg * kPage;
    u.first = row0 + (pos0 - start);
    u.r0 = lane / Tl::PAIRS;
    u.rotated = p < rot_pairs;
    u.e0 = (u.rotated ? p : 2 * rot_pairs + (p - rot_pairs)) * Tl::VE;
    u.e1 = u.e0 + (u.rotated ? rot_pairs : Tl::PAIRS - rot_pairs) * Tl::VE;

    const int nq = a.q ? a.n_heads : 0, nkv = a.pool.n_kv_heads, tiles = nq + 2 * nkv;
    auto load = [&](Tl& t, int tile) {
        if (tile < nq) t.load((const T*)a.q + (int64_t)tile * HD, a.q_stride, u);
        else if (tile < nq + nkv) t.load((const T*)a.k + (int64_t)(tile - nq) * HD, a.k_stride, u);
        else t.load((const T*)a.v + (int64_t)(tile - nq - nkv) * HD, a.v_stride, u);
    };
    const int step = gridDim.y * kWarps;
    int tile = blockIdx.y * kWarps + warp;
    Tl now;
    if (tile < tiles) load(now, tile);
    const int page = a.block_tables[(int64_t)b * a.max_pages + pg];
    const bool in_pool = page >= 0 && page < a.pool.n_pages;
    if (!in_pool && blockIdx.y == 0 && threadIdx.x == 0) flag_error(a.err, kErrBadContext);
    const int64_t block0 = ((int64_t)page * a.pool.n_layers + a.layer) * nkv;
    // the scale that a tile's block has so far, fetched with the tile
    auto scale_of = [&](int tile) { return tile < nq + nkv ? a.pool.k_scale + block0 + (tile - nq) : a.pool.v_scale + block0 + (tile - nq - nkv); };
    auto before_of = [&](int tile) { return u.slot0 && in_pool && tile >= nq && tile < tiles ? *scale_of(tile) : 0.0f; };
    float before = before_of(tile);
    if constexpr (ROT != kNone) {
        const int half = a.rot_dim / 2;
        for (int i = threadIdx.x * 4; i < u.n * half; i += blockDim.x * 4) {
            const int r = i / half, d = i % half;
            const int64_t at = (int64_t)(pos0 + r) * half + d;
            *reinterpret_cast<float4*>(&s_cos[r][d]) = *reinterpret_cast<const float4*>(a.rope_cos + at);
            *reinterpret_cast<float4*>(&s_sin[r][d]) = *reinterpret_cast<const float4*>(a.rope_sin + at);
        }
        __syncthreads();
    }

    while (tile < tiles) {
        __syncwarp();  // rows that repeat the last token are read before that is written in place
        if (tile < nq) {
            now.template turn<ROT, false>((T*)a.q_out + (int64_t)tile * HD, a.q_out_stride, u, s_cos, s_sin);
        } else if (tile < nq + nkv) {
            const int head = tile - nq;
            const float top = now.template turn<ROT, true>(a.k_out ? (T*)a.k_out + (int64_t)head * HD : nullptr, a.k_out_stride, u, s_cos, s_sin);
            now.forget_derived();
            if (in_pool)
                now.template append<ROT>(top, before, scale_of(tile), a.pool.k + (block0 + head) * (kPage * HD), u, s_cos, s_sin);
        } else if (in_pool) {
            const int head = tile - nq - nkv;
            const float top = now.template turn<kNone, true>(nullptr, 0, u, s_cos, s_sin);
            now.forget_derived();
            now.template append<kNone>(top, before, scale_of(tile), a.pool.v + (block0 + head) * (kPage * HD), u, s_cos, s_sin);
        }
        tile += step;
        if (tile < tiles) load(now, tile);
        before = before_of(tile);
    }
}

template <typename T, int HD>
cudaError_t launch_hd(const Kv8AppendArgs& a, dim3 grid, cudaStream_t s) {
    const dim3 block(kWarps * 32);
    if (!a.rot_dim) return launch_ex(kv8_append_kernel<T, HD, kNone>, grid, block, 0, s, 1, a);
    if (a.rope_layout == 0) return launch_ex(kv8_append_kernel<T, HD, kNeighbours>, grid, block, 0, s, 1, a);
    return launch_ex(kv8_append_kernel<T, HD, kHalves>, grid, block, 0, s, 1, a);
}

template <typename T>
cudaError_t launch_t(const Kv8AppendArgs& a, dim3 grid, cudaStream_t s) {
    return a.pool.head_dim == 64 ? launch_hd<T, 64>(a, grid, s) : launch_hd<T, 128>(a, grid, s);
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t s) {
    // All heads of a unit to one CTA where units alone fill the device, else as many CTAs as it
    // has tiles for.
    const int tiles = (a.q ? a.n_heads : 0) + 2 * a.pool.n_kv_heads, units = a.T / kPage + 2 * a.B;
    const int most = (tiles + kWarps - 1) / kWarps;
    const dim3 grid(units, std::min(most, std::max(1, kFill * 148 / units)));
    count_launch();
    if (a.dtype == kF32) return launch_t<float>(a, grid, s);
    if (a.dtype == kBF16) return launch_t<__nv_bfloat16>(a, grid, s);
    return launch_t<__half>(a, grid, s);
}

}  // namespace nitro
