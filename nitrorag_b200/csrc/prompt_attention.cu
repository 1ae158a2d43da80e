// Causal attention over packed prompts on the 5th-generation tensor cores
// (nr_prompt_attention).
//
// One CTA per two 128-row query tiles that read the same keys: two heads of one group on the
// same tokens where the group is even, else 256 consecutive tokens of one head.  Keys are
// taken 128 at a time:
//
//   warp 8     one thread copies Q once and K, V blocks into two-stage rings (TMA, 128-byte
//              swizzle, 64 dims to a box);
//   warp 9     one thread issues S_i = Q_i K^T into tensor memory and O_i += P_i V;
//   warps 0-3, 4-7   the softmax of tile 0 and of tile 1, one thread per query row: S row to
//              registers, running maximum, P = exp2(S - m) in the inputs' type written back
//              over S, from where it is the A operand of the second product.
//
// While one tile's softmax runs, the tensor cores work on the other tile.  S_i(j+1) is issued
// behind O_i += P_i(j) V(j) by the same thread, so it may take P's place, and a softmax warp
// that sees S_i(j+1) knows O_i complete: it rescales O_i in tensor memory itself, and only
// when the row's maximum has grown by 2^8 (P in bf16 or fp16 loses nothing by being up to
// 256), which after the first blocks hardly ever happens.
//
// P is rounded to the inputs' type for the second product, as its operands must have one
// type; the sum of a row is taken in fp32 over the unrounded values.
//
// The rows of a block behind a sequence's last key belong to other sequences and may hold
// anything.  As keys they are masked; as values 0 * NaN would be NaN, so the second product
// stops at the next multiple of 16 keys and the up to 15 rows left are set to zero in shared
// memory.
//
// Every wait is bounded; a CTA whose wait gave up sets the error flag and writes nothing
// more.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"
#include "tc_common.cuh"

namespace nitro {

namespace {

constexpr int kTile = 128;              // query rows of a tile, keys of a block
constexpr int kBox = kTile * 128;       // bytes of 128 rows x 64 dims
constexpr int kThreads = 10 * 32;
constexpr int kStages = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;

template <int HD>
constexpr int smem_bytes() { return (2 + 2 * kStages) * (HD / 64) * kBox + 1024; }

// Shared-memory matrix descriptor with 128-byte swizzle: 8-row groups 1024 bytes apart.
// K-major (rows of 64 K elements): lbo unused.  MN-major (64 N elements to a row of K): lbo
// is the distance of the next 64 N elements.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 | (uint64_t)(1024u >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// D fp32, A and B of one 16-bit type, A K-major, B K-major or (b_mn) MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc16(int N, bool b_mn) {
    const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// D (tensor memory) += A (tensor memory, 16 K elements = 8 columns) B (shared memory).
__device__ __forceinline__ void umma_tmem_a(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(head), "r"(row), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// Columns behind `limit` of 32 scores to -inf.
__device__ __forceinline__ void mask_row(uint32_t* v, int limit) {
#pragma unroll
    for (int k = 0; k < 32; k++)
        if (k > limit) v[k] = 0xff800000u;
}

struct Barriers {
    uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t s_full[2], p_full[2], o_full[2], done;
};

// PAIR: the two tiles are heads 2y, 2y + 1 of the same tokens; else tokens r and r + 128.
template <typename T, int HD, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, PromptAttnArgs a, int n_units) {
    constexpr int BOXES = HD / 64, W = PAIR ? kTile : 2 * kTile;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Barriers bar;
    __shared__ uint32_t tmem_slot;
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sq = smem;                                   // [tile][box]
    uint8_t* sk = sq + 2 * BOXES * kBox;                  // [stage][box]
    uint8_t* sv = sk + kStages * BOXES * kBox;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    grid_dependents_launch();

    // heads of one tile side by side (they share keys in L2), later tiles (more keys) first
    const int ny = PAIR ? a.n_heads / 2 : a.n_heads;
    const int unit = n_units - 1 - (int)(blockIdx.x / ny);
    const int head0 = (int)(blockIdx.x % ny) * (PAIR ? 2 : 1);
    const int kvh = head0 / (a.n_heads / a.n_kv_heads);
    const int* cu_k = a.cu_k ? a.cu_k : a.cu_q;
    const int b = seq_of_unit<W, 1>(a.cu_q, a.B, unit, lane);
    const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = cu_k[b], k1 = cu_k[b + 1];
    const int tile = unit - (q0 / W + b);
    if (tile < 0 || q0 == q1) return;
    if (q0 < 0 || q1 < q0 || q1 > a.Tq || k0 < 0 || k1 < k0 || k1 > a.Tk) {
        if (tile == 0 && threadIdx.x == 0) flag_error(a.err, kErrBadContext);
        return;
    }
    if ((int64_t)tile * W >= q1 - q0) return;
    const int off = (k1 - k0) - (q1 - q0);                // query r sees keys 0 .. r + off
    auto head = [&](int i) { return head0 + (PAIR ? i : 0); };
    auto row0 = [&](int i) { return tile * W + (PAIR ? 0 : i * kTile); };
    auto blocks_of = [&](int i) {
        const int rows = min(kTile, q1 - q0 - row0(i));
        const int keys = rows > 0 ? max(0, row0(i) + rows + off) : 0;  // all that the tile's last row sees
        return (keys + kTile - 1) / kTile;
    };
    const int blocks0 = blocks_of(0), blocks1 = blocks_of(1);
    const int n_blocks = max(blocks0, blocks1);

    if (warp == 9) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 1);
#pragma unroll
        for (int s = 0; s < kStages; s++) {
            mbar_init(&bar.k_full[s], 1);
            mbar_init(&bar.k_empty[s], 1);
            mbar_init(&bar.v_full[s], 1);
            mbar_init(&bar.v_empty[s], 1);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], kTile);
            mbar_init(&bar.o_full[i], 1);
        }
        mbar_init(&bar.done, 1);
        fence_barrier_init();
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    auto t_s = [&](int i) { return tmem + 128 * i; };
    auto t_o = [&](int i) { return tmem + 256 + HD * i; };

    if (warp == 8) {
        if (lane == 0 && n_blocks > 0) {
            mbar_arrive_expect_tx(&bar.q_full, 2 * BOXES * kBox);
            for (int i = 0; i < 2; i++)
                for (int x = 0; x < BOXES; x++)  // an absent second tile reads rows of others, unused
                    tma_load(sq + (i * BOXES + x) * kBox, &map_q, 64 * x, head(i), q0 + row0(i), &bar.q_full);
            int k_sent = 0, v_sent = 0;
            for (int j = 0; j < n_blocks; j++) {
                const int s = j % kStages;
                const uint32_t parity = (j / kStages - 1) & 1;
                if (j >= kStages && !mbar_wait(&bar.k_empty[s], parity, a.err)) break;
                mbar_arrive_expect_tx(&bar.k_full[s], BOXES * kBox);
                for (int x = 0; x < BOXES; x++)
                    tma_load(sk + (s * BOXES + x) * kBox, &map_k, 64 * x, kvh, k0 + j * kTile, &bar.k_full[s]);
                k_sent = j + 1;
                if (j >= kStages && !mbar_wait(&bar.v_empty[s], parity, a.err)) break;
                mbar_arrive_expect_tx(&bar.v_full[s], BOXES * kBox);
                for (int x = 0; x < BOXES; x++)
                    tma_load(sv + (s * BOXES + x) * kBox, &map_v, 64 * x, kvh, k0 + j * kTile, &bar.v_full[s]);
                v_sent = j + 1;
            }
            // no copy outlives the CTA, also when a wait gave up
            mbar_wait(&bar.q_full, 0, a.err);
            for (int j = max(0, k_sent - kStages); j < k_sent; j++) mbar_wait(&bar.k_full[j % kStages], (j / kStages) & 1, a.err);
            for (int j = max(0, v_sent - kStages); j < v_sent; j++) mbar_wait(&bar.v_full[j % kStages], (j / kStages) & 1, a.err);
        }
    } else if (warp == 9) {
        auto issue_s = [&](int i, int j) {  // S_i = Q_i K(j)^T
            if (lane == 0) {
#pragma unroll
                for (int x = 0; x < BOXES; x++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        umma_bf16(t_s(i), desc_sw128(smem_addr(sq + (i * BOXES + x) * kBox) + 32 * k, 16),
                                  desc_sw128(smem_addr(sk + ((j % kStages) * BOXES + x) * kBox) + 32 * k, 16),
                                  idesc16<T>(kTile, false), x + k > 0);
                umma_commit(&bar.s_full[i]);
                // the last of the block's readers frees it
                if (i == 1 || j >= blocks1) umma_commit(&bar.k_empty[j % kStages]);
            }
        };
        bool ok = n_blocks > 0 && mbar_wait(&bar.q_full, 0, a.err) && mbar_wait(&bar.k_full[0], 0, a.err);
        tc_fence_after();
        if (ok)
            for (int i = 0; i < 2; i++)
                if ((i ? blocks1 : blocks0) > 0) issue_s(i, 0);
        for (int j = 0; j < n_blocks && ok; j++) {
            const int s = j % kStages;
            const uint32_t parity = (j / kStages) & 1;
            ok = mbar_wait(&bar.v_full[s], parity, a.err);
            // values behind the last key: zero up to a multiple of 16 rows
            const int left = k1 - k0 - j * kTile;
            if (ok && left < kTile && left % 16) {
                for (int e = lane; e < (16 - left % 16) * 8 * BOXES; e += 32) {
                    const int x = e / (8 * (16 - left % 16)), in = e % (8 * (16 - left % 16));
                    *reinterpret_cast<uint4*>(sv + (s * BOXES + x) * kBox + left * 128 + in * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            __syncwarp();
            for (int i = 0; i < 2 && ok; i++) {
                if (j >= (i ? blocks1 : blocks0)) continue;
                ok = mbar_wait(&bar.p_full[i], j & 1, a.err);
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
                    const int steps = (min(left, kTile) + 15) / 16;
                    const uint64_t dv = desc_sw128(smem_addr(sv + s * BOXES * kBox), kBox);
                    for (int k = 0; k < steps; k++)  // 16 keys = 2048 bytes of values
                        umma_tmem_a(t_o(i), t_s(i) + 8 * k, dv + (uint64_t)(k * (2048 >> 4)), idesc16<T>(HD, true), j > 0 || k > 0);
                    if (i == 1 || j >= blocks1) umma_commit(&bar.v_empty[s]);
                }
                if (j + 1 < (i ? blocks1 : blocks0)) {
                    ok = mbar_wait(&bar.k_full[(j + 1) % kStages], ((j + 1) / kStages) & 1, a.err);
                    if (ok) issue_s(i, j + 1);
                } else if (lane == 0) {
                    umma_commit(&bar.o_full[i]);
                }
            }
        }
        if (lane == 0 && !ok && n_blocks > 0) {  // a wait gave up: let the products in flight end
            umma_commit(&bar.done);
            mbar_wait(&bar.done, 0, a.err);
        }
        __syncwarp();
    } else {
        const int i = warp >> 2;                          // tile
        const int blocks = i ? blocks1 : blocks0, first = row0(i);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
        const uint32_t ts = t_s(i) + lanes, to = t_o(i) + lanes;
        const int r = first + (warp & 3) * 32 + lane;   // row within the sequence
        const float scale = kLog2e * rsqrtf((float)HD);
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < blocks; j++) {
            ok = __all_sync(0xffffffffu, mbar_wait(&bar.s_full[i], j & 1, a.err));
            if (!ok) break;
            tc_fence_after();
            const int limit = r + off - j * kTile;        // last column this row sees
            const bool edge = j * kTile + kTile - 1 > first + off;
            // S is read twice, for the maximum and for the weights: tensor memory is fast, and a
            // whole row would not leave the registers to overlap anything
            uint32_t x[2][32];
            float top = -INFINITY;
            tmem_ld32_async(ts, x[0]);
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                uint32_t* v = x[(c >> 5) & 1];
                tmem_wait_ld();
                tmem_regs_ready(v);
                tmem_ld32_async(ts + (c + 32) % kTile, x[((c >> 5) + 1) & 1]);
                if (edge) mask_row(v, limit - c);
                float t[2] = {__uint_as_float(v[0]), __uint_as_float(v[1])};
#pragma unroll
                for (int k = 2; k < 32; k += 4) {
                    t[0] = fmaxf(t[0], fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 1])));
                    if (k + 2 < 32) t[1] = fmaxf(t[1], fmaxf(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3])));
                }
                top = fmaxf(top, fmaxf(t[0], t[1]));
            }
            top *= scale;
            const bool grows = top > m + kLazy;
            if (__any_sync(0xffffffffu, grows)) {
                const float corr = !grows ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - top);
                if (grows) m = top;
                l *= corr;
                if (j > 0) {
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tmem_ld32_async(to + c, o);
                        tmem_wait_ld();
                        tmem_regs_ready(o);
#pragma unroll
                        for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                        tmem_st32(to + c, o);
                    }
                }
            }
            const float shift = m == -INFINITY ? 0.0f : -m;
            const unsigned long long scale2 = pack2(__float_as_uint(scale), __float_as_uint(scale));
            const unsigned long long shift2 = pack2(__float_as_uint(shift), __float_as_uint(shift));
            unsigned long long sum[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                uint32_t* v = x[(c >> 5) & 1];
                tmem_wait_ld();
                tmem_regs_ready(v);
                if (c + 32 < kTile) tmem_ld32_async(ts + c + 32, x[((c >> 5) + 1) & 1]);
                if (edge) mask_row(v, limit - c);
                uint32_t p[16];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    uint32_t y0, y1;
                    unpack2(fma2(pack2(v[k], v[k + 1]), scale2, shift2), y0, y1);
                    const float e0 = exp2_fast(__uint_as_float(y0)), e1 = exp2_fast(__uint_as_float(y1));
                    sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], pack2(__float_as_uint(e0), __float_as_uint(e1)));
                    p[k / 2] = pack16<T>(e0, e1);
                }
                tmem_st16(ts + c / 2, p);
            }
            {
                uint32_t a0, a1;
                unpack2(add2(sum[0], sum[1]), a0, a1);
                l += __uint_as_float(a0) + __uint_as_float(a1);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bar.p_full[i]);
        }
        if (ok && blocks > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(&bar.o_full[i], 0, a.err));
            tc_fence_after();
        }
        if (ok && first < q1 - q0) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* out = (T*)a.out + (int64_t)(q0 + r) * a.out_stride + (int64_t)head(i) * HD;
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (blocks > 0) {
                    tmem_ld32_async(to + c, o);
                    tmem_wait_ld();
                    tmem_regs_ready(o);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; k++) o[k] = 0;
                }
                if (r >= q1 - q0) continue;
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)  // a row that sees no key has l = 0 and whatever O: select, do not multiply
                        w[e] = l == 0.0f ? 0u : pack16<T>(__uint_as_float(o[k + 2 * e]) * inv, __uint_as_float(o[k + 2 * e + 1]) * inv);
                    *reinterpret_cast<uint4*>(out + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeFn)p;
    }();
    return fn;
}

// Rows of `heads` heads as boxes of 128 rows x 64 dims of one head.
bool encode(CUtensorMap* m, int dtype, const void* p, int64_t stride, int rows, int heads, int hd) {
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, 1, kTile}, ones[3] = {1, 1, 1};
    return encode_fn()(m, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                       const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, bool PAIR>
cudaError_t launch_tiles(const PromptAttnArgs& a, cudaStream_t s) {
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is set
    int dev = 0;
    cudaError_t rc = cudaGetDevice(&dev);
    if (rc != cudaSuccess) return rc;
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        rc = cudaFuncSetAttribute(prompt_attn_kernel<T, HD, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<HD>());
        if (rc != cudaSuccess) return rc;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev);
    }
    if (!encode_fn()) return cudaErrorNotSupported;
    CUtensorMap mq, mk, mv;
    if (!encode(&mq, a.dtype, a.q, a.q_stride, a.Tq, a.n_heads, HD) ||
        !encode(&mk, a.dtype, a.k, a.k_stride, a.Tk, a.n_kv_heads, HD) ||
        !encode(&mv, a.dtype, a.v, a.v_stride, a.Tk, a.n_kv_heads, HD))
        return cudaErrorInvalidValue;
    const int units = a.Tq / (PAIR ? kTile : 2 * kTile) + a.B;
    const unsigned grid = (unsigned)units * (unsigned)(PAIR ? a.n_heads / 2 : a.n_heads);
    count_launch();
    return launch_ex(prompt_attn_kernel<T, HD, PAIR>, dim3(grid), dim3(kThreads), smem_bytes<HD>(), s, 1, mq, mk, mv, a, units);
}

template <typename T, int HD>
cudaError_t launch_hd(const PromptAttnArgs& a, cudaStream_t s) {
    return a.n_heads / a.n_kv_heads % 2 ? launch_tiles<T, HD, false>(a, s) : launch_tiles<T, HD, true>(a, s);
}

}  // namespace

cudaError_t launch_prompt_attention(const PromptAttnArgs& a, cudaStream_t s) {
    if (a.dtype == kBF16) return a.head_dim == 64 ? launch_hd<__nv_bfloat16, 64>(a, s) : launch_hd<__nv_bfloat16, 128>(a, s);
    return a.head_dim == 64 ? launch_hd<__half, 64>(a, s) : launch_hd<__half, 128>(a, s);
}

}  // namespace nitro
