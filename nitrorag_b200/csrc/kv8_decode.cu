// Decode attention over e4m3 pages (nr_paged_attention_decode_kv8).
//
// One CTA per (sequence, head): each warp takes every fourth page with its own running
// maximum, sum and output (lane l holds dims l, l + 32, ...), joined through shared memory.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"

namespace nitro {

namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ float e4m3_f32(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32) kv8_decode_kernel(Kv8DecodeArgs a) {
    constexpr int D = HD / 32;
    __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x, b = blockIdx.y;
    grid_dependency_wait();
    grid_dependents_launch();
    int ctx = a.ctx_lens[b];
    if (ctx < 0 || ctx > (int64_t)a.max_pages * kPage) {
        if (threadIdx.x == 0) flag_error(a.err, kErrBadContext);
        ctx = ctx < 0 ? 0 : a.max_pages * kPage;
    }
    const int nkv = a.pool.n_kv_heads, kvh = h / (a.n_heads / nkv);
    const T* q = (const T*)a.q + ((int64_t)b * a.n_heads + h) * HD;
    float qv[D], o[D], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < D; i++) {
        qv[i] = to_f32(q[lane + 32 * i]) * rsqrtf((float)HD);
        o[i] = 0.0f;
    }
    for (int pg = warp; pg * kPage < ctx; pg += kWarps) {
        const int page = a.block_tables[(int64_t)b * a.max_pages + pg];
        if (page < 0 || page >= a.pool.n_pages) {
            if (lane == 0) flag_error(a.err, kErrBadContext);
            continue;
        }
        const int64_t block = ((int64_t)page * a.pool.n_layers + a.layer) * nkv + kvh;
        const float ks = a.pool.k_scale[block], vs = a.pool.v_scale[block];
        for (int r = 0; r < min(kPage, ctx - pg * kPage); r++) {
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < D; i++) x += qv[i] * e4m3_f32(a.pool.k[(block * kPage + r) * HD + lane + 32 * i]);
            x = warp_sum(x) * ks;
            const float mn = fmaxf(m, x);
            const float c = m == -INFINITY ? 0.0f : expf(m - mn), p = x == -INFINITY ? 0.0f : expf(x - mn);
            m = mn;
            l = l * c + p;
#pragma unroll
            for (int i = 0; i < D; i++)
                o[i] = o[i] * c + p * vs * e4m3_f32(a.pool.v[(block * kPage + r) * HD + lane + 32 * i]);
        }
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int i = 0; i < D; i++) s_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float mm = -INFINITY;
    for (int w = 0; w < kWarps; w++) mm = fmaxf(mm, s_m[w]);
    for (int d = threadIdx.x; d < HD; d += blockDim.x) {
        float sum = 0.0f, acc = 0.0f;
        for (int w = 0; w < kWarps; w++) {
            const float c = s_m[w] == -INFINITY ? (s_l[w] != s_l[w] ? s_l[w] : 0.0f) : expf(s_m[w] - mm);
            sum += c * s_l[w];
            acc += c * s_o[w][d];
        }
        ((T*)a.out)[((int64_t)b * a.n_heads + h) * HD + d] = from_f32<T>(sum == 0.0f ? 0.0f : acc / sum);
    }
}

template <typename T>
cudaError_t launch_t(const Kv8DecodeArgs& a, cudaStream_t s) {
    const dim3 grid(a.n_heads, a.B);
    if (a.pool.head_dim == 64) return launch_ex(kv8_decode_kernel<T, 64>, grid, dim3(kWarps * 32), 0, s, 1, a);
    return launch_ex(kv8_decode_kernel<T, 128>, grid, dim3(kWarps * 32), 0, s, 1, a);
}

}  // namespace

size_t kv8_decode_workspace_bytes(int, int, int, int, int) { return 256; }

cudaError_t launch_kv8_decode(const Kv8DecodeArgs& a, cudaStream_t s) {
    count_launch();
    if (a.dtype == kF32) return launch_t<float>(a, s);
    if (a.dtype == kBF16) return launch_t<__nv_bfloat16>(a, s);
    return launch_t<__half>(a, s);
}

}  // namespace nitro
