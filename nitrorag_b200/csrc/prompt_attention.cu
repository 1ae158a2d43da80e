// Causal attention over packed prompts (nr_prompt_attention).
//
// One warp per (query row, head): lane l holds dims l, l + 32, ...; running maximum and sum.
#include <cuda_runtime.h>

#include <cmath>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"

namespace nitro {

namespace {

template <typename T, int HD>
__global__ void __launch_bounds__(128) prompt_attn_kernel(PromptAttnArgs a) {
    constexpr int D = HD / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    grid_dependents_launch();
    const int* cu_k = a.cu_k ? a.cu_k : a.cu_q;
    const int h = blockIdx.y, kvh = h / (a.n_heads / a.n_kv_heads);
    const int u = blockIdx.x;
    const int b = seq_of_unit<128, 1>(a.cu_q, a.B, u, lane);
    const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = cu_k[b], k1 = cu_k[b + 1];
    const int tile = u - (q0 / 128 + b);
    if (tile < 0 || q0 == q1) return;
    if (q0 < 0 || q1 < q0 || q1 > a.Tq || k0 < 0 || k1 < k0 || k1 > a.Tk) {
        if (tile == 0 && threadIdx.x == 0) flag_error(a.err, kErrBadContext);
        return;
    }
    for (int i = warp; i < 128; i += 4) {
        const int64_t r = (int64_t)q0 + tile * 128 + i;
        if (r >= q1) break;
        const T* q = (const T*)a.q + r * a.q_stride + (int64_t)h * HD;
        float qv[D], o[D], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int d = 0; d < D; d++) {
            qv[d] = to_f32(q[lane + 32 * d]) * rsqrtf((float)HD);
            o[d] = 0.0f;
        }
        const int seen = (int)(r - q0) + 1 + (k1 - k0) - (q1 - q0);
        for (int j = 0; j < seen; j++) {
            const T* k = (const T*)a.k + (int64_t)(k0 + j) * a.k_stride + (int64_t)kvh * HD;
            const T* v = (const T*)a.v + (int64_t)(k0 + j) * a.v_stride + (int64_t)kvh * HD;
            float x = 0.0f;
#pragma unroll
            for (int d = 0; d < D; d++) x += qv[d] * to_f32(k[lane + 32 * d]);
            x = warp_sum(x);
            const float mn = fmaxf(m, x), c = expf(m - mn), p = expf(x - mn);
            m = mn;
            l = l * c + p;
#pragma unroll
            for (int d = 0; d < D; d++) o[d] = o[d] * c + p * to_f32(v[lane + 32 * d]);
        }
#pragma unroll
        for (int d = 0; d < D; d++)
            ((T*)a.out)[r * a.out_stride + (int64_t)h * HD + lane + 32 * d] = from_f32<T>(l == 0.0f ? 0.0f : o[d] / l);
    }
}

template <typename T>
cudaError_t launch_t(const PromptAttnArgs& a, cudaStream_t s) {
    const dim3 grid(a.Tq / 128 + a.B, a.n_heads);
    if (a.head_dim == 64) return launch_ex(prompt_attn_kernel<T, 64>, grid, dim3(128), 0, s, 1, a);
    return launch_ex(prompt_attn_kernel<T, 128>, grid, dim3(128), 0, s, 1, a);
}

}  // namespace

cudaError_t launch_prompt_attention(const PromptAttnArgs& a, cudaStream_t s) {
    count_launch();
    return a.dtype == kBF16 ? launch_t<__nv_bfloat16>(a, s) : launch_t<__half>(a, s);
}

}  // namespace nitro
