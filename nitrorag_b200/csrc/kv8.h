// Host-side launchers of the kernels behind the 8-bit K/V pages and the operators that are
// used with them (no counterpart in the reference).
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace nitro {

// NR_DTYPE_* of include/nitro_engine.h
enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline int dtype_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

// Codes [page][layer][kv_head][16][head_dim] (e4m3), scales [page][layer][kv_head].
struct Kv8Pool {
    uint8_t* k = nullptr;
    uint8_t* v = nullptr;
    float* k_scale = nullptr;
    float* v_scale = nullptr;
    int n_pages = 0, n_layers = 0, n_kv_heads = 0, head_dim = 0;
};

struct Kv8AppendArgs {
    Kv8Pool pool;
    const void* q = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    void* q_out = nullptr;
    void* k_out = nullptr;
    int64_t q_stride = 0, k_stride = 0, v_stride = 0, q_out_stride = 0, k_out_stride = 0;
    const int* cu_seqlens = nullptr;
    const int* start_pos = nullptr;
    const int* block_tables = nullptr;
    const float* rope_cos = nullptr;
    const float* rope_sin = nullptr;
    int dtype = 0, B = 0, T = 0, n_heads = 0, max_pages = 0, layer = 0, rope_len = 0, rot_dim = 0, rope_layout = 0;
    int* err = nullptr;
};
cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t s);

struct Kv8DecodeArgs {
    Kv8Pool pool;
    const void* q = nullptr;
    void* out = nullptr;
    const int* block_tables = nullptr;
    const int* ctx_lens = nullptr;
    void* workspace = nullptr;
    int dtype = 0, layer = 0, max_pages = 0, B = 0, n_heads = 0;
    int* err = nullptr;
};
size_t kv8_decode_workspace_bytes(int B, int n_heads, int n_kv_heads, int head_dim, int max_pages);
cudaError_t launch_kv8_decode(const Kv8DecodeArgs& a, cudaStream_t s);

struct PromptAttnArgs {
    const void* q = nullptr;
    const void* k = nullptr;
    const void* v = nullptr;
    void* out = nullptr;
    int64_t q_stride = 0, k_stride = 0, v_stride = 0, out_stride = 0;
    const int* cu_q = nullptr;
    const int* cu_k = nullptr;
    int dtype = 0, B = 0, Tq = 0, Tk = 0, n_heads = 0, n_kv_heads = 0, head_dim = 0;
    int* err = nullptr;
};
cudaError_t launch_prompt_attention(const PromptAttnArgs& a, cudaStream_t s);

struct LogprobArgs {
    const void* logits = nullptr;
    int dtype = 0;
    int64_t row_stride = 0;
    int M = 0, V = 0, top_k = 0;
    const int* targets = nullptr;
    float* target_logprob = nullptr;
    float* entropy = nullptr;
    float* top_logprob = nullptr;
    int* top_ids = nullptr;
};
cudaError_t launch_token_logprobs(const LogprobArgs& a, cudaStream_t s);

}  // namespace nitro
