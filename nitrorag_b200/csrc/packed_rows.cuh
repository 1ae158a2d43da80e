// Small device helpers of the kernels over packed rows and 8-bit pages: element types as
// fp32, and finding the sequence a unit of work belongs to.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace nitro {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Units of work of packed sequences: sequence b owns the units from cu[b]/W + PER*b up to
// the next sequence's first.  A sequence of n rows has floor(n/W) + PER of them at least,
// which holds its ceil(n/W) tiles (PER = 1) or the W-token pages it touches from any start
// (at most floor(n/W) + 2: PER = 2), so T/W + PER*B units cover every sequence without the
// host knowing the lengths.  Returns the last sequence whose first unit is not behind u
// (0 if none): every lane of the warp probes one of 32 points of the interval left.
template <int W, int PER>
__device__ __forceinline__ int seq_of_unit(const int* cu, int B, int u, int lane) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int i = lo + lane * step;
        const bool at = i < hi && cu[i] / W + PER * i <= u;
        const int k = max(__popc(__ballot_sync(0xffffffffu, at)) - 1, 0);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

__device__ __forceinline__ void flag_error(int* err, int code) {
    if (err) atomicCAS(err, 0, code);
}

}  // namespace nitro
