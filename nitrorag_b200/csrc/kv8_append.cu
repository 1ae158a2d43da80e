// Append of rotated keys and values to e4m3 pages (nr_kv8_append).
//
// One unit of work is the part of one page that a sequence's new tokens fall into, at most
// 16 tokens; one warp takes one head of one unit (a head of q, k or v): the whole 16 x
// head_dim tile sits in the warp's registers, so the rotation, the block's maximum, the
// scale and the codes come from one read of the input.
//
// Scale of a block: the smallest 2^e with |x| <= 448 * 2^e (448 is the largest e4m3 value).
// With |x|max = 1.m * 2^E and 448 = 1.75 * 2^8 that is e = E - 8, one more if 1.m > 1.75:
// read off the float's bits.  e4m3 keeps its relative precision over 2^14, so rounding the
// scale up to a power of two loses no accuracy, and dividing by it is exact: a block that
// grows token by token ends with the codes it would have got at once (but for values that
// fall below the normal range), and the older codes are not rounded again and again.
// The maximum is taken over the bits of |x| as unsigned numbers, in which infinities and
// NaNs are largest: they reach the scale, which becomes NaN.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"

namespace nitro {

namespace {

constexpr int kWarps = 8;

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
    static __device__ __forceinline__ void load(const T* p, float* v) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
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

// A row's vectors are taken in pairs so that a lane holds both elements of every rotation
// pair: (j, j + half the rotated vectors) in the rotated part, the same split of the rest.
template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32) kv8_append_kernel(Kv8AppendArgs a) {
    constexpr int VE = Vec<T>::N;
    constexpr int PAIRS = HD / (2 * VE);       // vector pairs in a row
    constexpr int ROWS = 32 / PAIRS;           // rows a warp covers at a time
    constexpr int STEPS = kPage / ROWS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    grid_dependents_launch();
    const int b = seq_of_unit<kPage, 2>(a.cu_seqlens, a.B, blockIdx.x, lane);
    const int row0 = a.cu_seqlens[b], row1 = a.cu_seqlens[b + 1], start = a.start_pos[b];
    const int j = (int)blockIdx.x - (row0 / kPage + 2 * b);
    if (j < 0 || row1 == row0) return;
    const int64_t end = (int64_t)start + row1 - row0;
    if (row0 < 0 || row1 < row0 || row1 > a.T || start < 0 || end > (int64_t)a.max_pages * kPage ||
        (a.rot_dim && end > a.rope_len)) {
        if (j == 0 && threadIdx.x == 0) flag_error(a.err, kErrBadContext);
        return;
    }
    const int pg = start / kPage + j;
    if ((int64_t)pg * kPage >= end) return;
    const int pos0 = max(start, pg * kPage), n = min((int)end, (pg + 1) * kPage) - pos0;
    const int slot0 = pos0 - pg * kPage;       // rows of the page that are there already
    const int64_t first = row0 + (pos0 - start);

    const int p = lane % PAIRS, r0 = lane / PAIRS;
    const int rot_pairs = a.rot_dim / (2 * VE);
    const bool rotated = p < rot_pairs;
    const int rest = PAIRS - rot_pairs;
    const int e0 = rotated ? p * VE : (2 * rot_pairs + (p - rot_pairs)) * VE;  // first elements of the two vectors
    const int e1 = e0 + (rotated ? rot_pairs : rest) * VE;

    const int nq = a.q ? a.n_heads : 0, nkv = a.pool.n_kv_heads;
    for (int tile = blockIdx.y * kWarps + warp; tile < nq + 2 * nkv; tile += gridDim.y * kWarps) {
        const bool is_q = tile < nq, is_v = tile >= nq + nkv;
        const int head = is_q ? tile : is_v ? tile - nq - nkv : tile - nq;
        const T* src = (const T*)(is_q ? a.q : is_v ? a.v : a.k) + (int64_t)head * HD;
        const int64_t ld = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;
        float x[STEPS][2][VE];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int r = s * ROWS + r0;
            if (r < n) {
                const T* row = src + (first + r) * ld;
                Vec<T>::load(row + e0, x[s][0]);
                Vec<T>::load(row + e1, x[s][1]);
            } else {
#pragma unroll
                for (int i = 0; i < VE; i++) x[s][0][i] = x[s][1][i] = 0.0f;
            }
        }
        if (!is_v && rotated) {
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int r = s * ROWS + r0;
                if (r >= n) continue;
                const int64_t t = (int64_t)(pos0 + r) * (a.rot_dim / 2);
                if (a.rope_layout == 1) {
#pragma unroll
                    for (int i = 0; i < VE; i += 4) {
                        const float4 c = *reinterpret_cast<const float4*>(a.rope_cos + t + e0 + i);
                        const float4 sn = *reinterpret_cast<const float4*>(a.rope_sin + t + e0 + i);
                        const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float x0 = x[s][0][i + k], x1 = x[s][1][i + k];
                            x[s][0][i + k] = __fsub_rn(__fmul_rn(x0, cc[k]), __fmul_rn(x1, ss[k]));
                            x[s][1][i + k] = __fadd_rn(__fmul_rn(x0, ss[k]), __fmul_rn(x1, cc[k]));
                        }
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int i = 0; i < VE; i += 4) {
                            const int64_t at = t + ((h ? e1 : e0) + i) / 2;
                            const float2 c = *reinterpret_cast<const float2*>(a.rope_cos + at);
                            const float2 sn = *reinterpret_cast<const float2*>(a.rope_sin + at);
                            const float cc[2] = {c.x, c.y}, ss[2] = {sn.x, sn.y};
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const float x0 = x[s][h][i + 2 * k], x1 = x[s][h][i + 2 * k + 1];
                                x[s][h][i + 2 * k] = __fsub_rn(__fmul_rn(x0, cc[k]), __fmul_rn(x1, ss[k]));
                                x[s][h][i + 2 * k + 1] = __fadd_rn(__fmul_rn(x0, ss[k]), __fmul_rn(x1, cc[k]));
                            }
                        }
                }
            }
        }
        if (!is_v && (is_q || a.k_out)) {
            T* dst = (T*)(is_q ? a.q_out : a.k_out) + (int64_t)head * HD;
            const int64_t lo = is_q ? a.q_out_stride : a.k_out_stride;
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int r = s * ROWS + r0;
                if (r < n) {
                    Vec<T>::store(dst + (first + r) * lo + e0, x[s][0]);
                    Vec<T>::store(dst + (first + r) * lo + e1, x[s][1]);
                }
            }
        }
        if (is_q) continue;
        const int page = a.block_tables[(int64_t)b * a.max_pages + pg];
        if (page < 0 || page >= a.pool.n_pages) {
            if (lane == 0) flag_error(a.err, kErrBadContext);
            continue;
        }
        uint32_t amax = 0;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int i = 0; i < VE; i++)
                amax = max(amax, max(__float_as_uint(x[s][0][i]) & 0x7fffffffu, __float_as_uint(x[s][1][i]) & 0x7fffffffu));
        amax = __reduce_max_sync(0xffffffffu, amax);
        const int64_t block = ((int64_t)page * a.pool.n_layers + a.layer) * nkv + head;
        float* scale_at = (is_v ? a.pool.v_scale : a.pool.k_scale) + block;
        uint8_t* codes = (is_v ? a.pool.v : a.pool.k) + block * (kPage * HD);
        float scale = block_scale(amax);
        if (slot0) {
            const float before = *scale_at;
            const bool grows = __float_as_uint(scale) > __float_as_uint(before);
            if (grows) {
                const float r = before / scale;
                for (int i = lane * 16; i < slot0 * HD; i += 32 * 16) {
                    uint4* c = reinterpret_cast<uint4*>(codes + i);
                    *c = recode(*c, r);
                }
            } else {
                scale = before;
            }
            __syncwarp();  // every lane has read the old scale
            if (grows && lane == 0) *scale_at = scale;
        } else if (lane == 0) {
            *scale_at = scale;
        }
        const float inv = 1.0f / scale;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int r = s * ROWS + r0;
            if (r < n) {
                Vec<T>::store_codes(codes + (slot0 + r) * HD + e0, x[s][0], inv);
                Vec<T>::store_codes(codes + (slot0 + r) * HD + e1, x[s][1], inv);
            }
        }
    }
}

template <typename T>
cudaError_t launch_t(const Kv8AppendArgs& a, dim3 grid, cudaStream_t s) {
    if (a.pool.head_dim == 64) return launch_ex(kv8_append_kernel<T, 64>, grid, dim3(kWarps * 32), 0, s, 1, a);
    return launch_ex(kv8_append_kernel<T, 128>, grid, dim3(kWarps * 32), 0, s, 1, a);
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t s) {
    const int tiles = (a.q ? a.n_heads : 0) + 2 * a.pool.n_kv_heads;
    const dim3 grid(a.T / kPage + 2 * a.B, (tiles + kWarps - 1) / kWarps);
    count_launch();
    if (a.dtype == kF32) return launch_t<float>(a, grid, s);
    if (a.dtype == kBF16) return launch_t<__nv_bfloat16>(a, grid, s);
    return launch_t<__half>(a, grid, s);
}

}  // namespace nitro
