// Token log probabilities, entropy and top alternatives (nr_token_logprobs).
//
// One CTA per row; statistics in two passes over the row, then one pass for each of the
// top_k entries (the largest key below the last one found).
#include <cuda_runtime.h>

#include <cmath>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"

namespace nitro {

namespace {

constexpr int kThreads = 1024;

// Ranks (value, id): larger value first, then smaller id; NaN below -inf.
__device__ __forceinline__ unsigned long long rank_key(float v, int id) {
    uint32_t u = __float_as_uint(v + 0.0f);
    u = v != v ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (0xffffffffu - (uint32_t)id);
}

template <typename F, typename V>
__device__ V block_reduce(V v, F f, V* tmp) {
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = tmp[0];
    for (int i = 1; i < kThreads / 32; i++) v = f(v, tmp[i]);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_kernel(LogprobArgs a) {
    __shared__ float tf[kThreads / 32];
    __shared__ unsigned long long tk[kThreads / 32];
    const int64_t row = blockIdx.x;
    grid_dependency_wait();
    grid_dependents_launch();
    const T* x = (const T*)a.logits + row * a.row_stride;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < a.V; i += kThreads) m = fmaxf(m, to_f32(x[i]));
    m = block_reduce(m, [](float p, float q) { return fmaxf(p, q); }, tf);
    float s = 0.0f, w = 0.0f;
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
        const float y = to_f32(x[i]) - m, e = expf(y);
        s += e;
        if (e != 0.0f) w += e * y;
    }
    auto add = [](float p, float q) { return p + q; };
    s = block_reduce(s, add, tf);
    w = block_reduce(w, add, tf);
    const float ls = logf(s);
    if (threadIdx.x == 0) {
        if (a.targets) {
            const int t = a.targets[row];
            a.target_logprob[row] = t < 0 || t >= a.V ? NAN : (to_f32(x[t]) - m) - ls;
        }
        if (a.entropy) a.entropy[row] = ls - w / s;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top_k; k++) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < a.V; i += kThreads) {
            const unsigned long long key = rank_key(to_f32(x[i]), i);
            if (key < last && key > best) best = key;
        }
        best = block_reduce(best, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; }, tk);
        last = best;
        if (threadIdx.x == 0) {
            const int id = (int)(0xffffffffu - (uint32_t)best);
            a.top_ids[row * a.top_k + k] = id;
            a.top_logprob[row * a.top_k + k] = (to_f32(x[id]) - m) - ls;
        }
    }
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, cudaStream_t s) {
    count_launch();
    if (a.dtype == kF32) return launch_ex(logprob_kernel<float>, dim3(a.M), dim3(kThreads), 0, s, 1, a);
    if (a.dtype == kBF16) return launch_ex(logprob_kernel<__nv_bfloat16>, dim3(a.M), dim3(kThreads), 0, s, 1, a);
    return launch_ex(logprob_kernel<__half>, dim3(a.M), dim3(kThreads), 0, s, 1, a);
}

}  // namespace nitro
