// Causal attention over packed prompts on the 5th-generation tensor cores
// (nr_prompt_attention).
//
// A CTA takes two 128-row query tiles that read the same keys (head_dim 128: two heads of a
// group on the same tokens where the group is even, else 256 consecutive tokens of one head)
// or one (head_dim 64, two CTAs to an SM).  Keys are taken 128 at a time:
//
//   copy warp      one thread copies Q once and K, V blocks into two-stage rings (TMA, 128-byte
//                  swizzle, 64 dims to a box);
//   product warp   one thread issues S_i = Q_i K^T into tensor memory and O_i += P_i V;
//   softmax        four warps for each tile, one thread per query row: S row to registers, running
//                  maximum, P = exp2(S - m) in the inputs' type written back over S, from
//                  where it is the A operand of the second product.
//
// While one tile's softmax runs, the tensor cores work on the other tile.  S_i(j+1) is issued
// behind O_i += P_i(j) V(j) by the same thread, so it may take P's place, and a softmax warp
// that sees S_i(j+1) knows O_i complete: it rescales O_i in tensor memory itself, and only
// when the row's maximum has grown by 2^8 (P in bf16 or fp16 loses nothing by being up to
// 256), which after the first blocks hardly ever happens.  So the weights of a block's first 64
// keys are taken from the old maximum while the new one is being found, and their product
// starts while the other 64 are computed.
//
// P is rounded to the inputs' type for the second product, as its operands must have one
// type; the sum of a row is taken in fp32 over the unrounded values.
//
// The rows of a block behind a sequence's last key belong to other sequences and may hold
// anything.  As keys they are masked; as values 0 * NaN would be NaN, so the second product
// stops at the next multiple of 16 keys and the up to 15 rows left are set to zero in shared
// memory.
//
// Measured: one prompt of 8192 tokens, 32 heads on 8, head_dim 128: 433 us, 1270 TFLOP/s of the
// causal half, 0.76 of the measured cuBLAS rate (sustained: 511 us, 0.78 of its sustained
// rate; the clock falls under the power limit, and variants that saved a tenth of the cycles
// saved no time).  Per 128-key step of both tiles the tensor cores need 2300 cycles (the first
// product 640, bound by reading both operands from shared memory, the second 512, twice), the
// special function unit 2100, a step takes 3000.  head_dim 64 has half the products for the
// same exponentials: 664 TFLOP/s at 8192 tokens, 32 heads on 8.  Tried and left: a product warp for each
// tile (their products interleave: 485 us), two threads to a row (497), exponentials partly by
// polynomial (437: the issue slots it takes are the ones that are short), S read twice
// instead of a row in registers (473).
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
// Registers a thread with two tiles: launched with 168 each (65536 / 384); the third warpgroup
// gives what the softmax needs to hold a row of S: 2 * 208 + 88 = 3 * 168.
constexpr int kRegsSoftmax = 208, kRegsOther = 88;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;
constexpr int kFirst = 64;              // keys of a block whose weights are handed over first

// What a CTA's tiles are: one of them; two heads of a group on the same tokens; two tiles of
// one head, 128 tokens apart.
enum Tiling { kOne, kHeads, kRows };
template <int HD, Tiling TILING>
struct Layout {
    static constexpr int kTiles = TILING == kOne ? 1 : 2;
    static constexpr int kRowsPerUnit = TILING == kRows ? 2 * kTile : kTile;
    static constexpr int kStages = TILING == kOne && HD == 128 ? 1 : 2;  // K and V blocks in flight
    static constexpr int kCopyWarp = 4 * kTiles, kMmaWarp = kCopyWarp + 1;
    // two tiles: three whole warpgroups (the last two warps idle) for the register split
    static constexpr int kThreads = TILING == kOne ? 6 * 32 : 12 * 32;
    static constexpr int kCtas = TILING == kOne ? 2 : 1;  // on an SM
    static constexpr uint32_t kTmem = TILING == kOne ? 256 : 512;
    static constexpr int kSmem = (kTiles + 2 * kStages) * (HD / 64) * kBox + 1024;
    static_assert(kTiles * (kTile + HD) <= (int)kTmem && kCtas * kTmem <= 512, "tensor memory");
};

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

// True in one lane of the (converged) warp.  Unlike a test of the lane number this lets the
// compiler keep the operands of the products issued under it in uniform registers: with
// `lane == 0` an issue took 120 cycles, twice as long as the product itself.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(head), "r"(row), "r"(smem_addr(bar))
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

// Columns behind `limit` of N scores to -inf.
template <int N>
__device__ __forceinline__ void mask_row(uint32_t* v, int limit) {
#pragma unroll
    for (int k = 0; k < N; k++)
        if (k > limit) v[k] = 0xff800000u;
}

template <int N>
__device__ __forceinline__ float max_row(const uint32_t* v) {
    float t[4];
#pragma unroll
    for (int k = 0; k < 4; k++) t[k] = __uint_as_float(v[k]);
#pragma unroll
    for (int k = 4; k + 1 < N; k += 2)
        t[(k >> 1) & 3] = fmaxf(t[(k >> 1) & 3], fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 1])));
    return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
}

// exp2(v * scale + shift) of N columns into tensor memory, rounded to T, their sum added to
// sum.
template <typename T, int N>
__device__ __forceinline__ void weights(const uint32_t* v, unsigned long long scale2, unsigned long long shift2,
                                        unsigned long long* sum, uint32_t tp) {
#pragma unroll
    for (int c = 0; c < N; c += 32) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
            uint32_t y0, y1;
            unpack2(fma2(pack2(v[c + k], v[c + k + 1]), scale2, shift2), y0, y1);
            const float e0 = exp2_fast(__uint_as_float(y0)), e1 = exp2_fast(__uint_as_float(y1));
            sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], pack2(__float_as_uint(e0), __float_as_uint(e1)));
            p[k / 2] = pack16<T>(e0, e1);
        }
        tmem_st16(tp + c / 2, p);
    }
}

// mbar_wait with a bound on the polls (of up to 1 us each): no clock is read, the code
// between two products stays short.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* err) {
#pragma unroll 1
    for (int n = 0; n < 4000000; n++)
        if (mbar_try_wait(bar, parity)) return true;
    flag_error(err, kErrWaitTimeout);
    return false;
}

struct Barriers {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t s_full[2], p_first[2], p_full[2], o_full[2], done;
};

template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int HD, Tiling TILING>
__global__ void __launch_bounds__(Layout<HD, TILING>::kThreads, Layout<HD, TILING>::kCtas)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, PromptAttnArgs a, int n_units) {
    using L = Layout<HD, TILING>;
    constexpr int BOXES = HD / 64, W = L::kRowsPerUnit, TILES = L::kTiles, kStages = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Barriers bar;
    __shared__ uint32_t tmem_slot;
    __shared__ int s_tile, s_q0, s_q1, s_k0, s_k1;
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sq = smem;                                   // [tile][box]
    uint8_t* sk = sq + TILES * BOXES * kBox;              // [stage][box]
    uint8_t* sv = sk + kStages * BOXES * kBox;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
        for (int i = 0; i < TILES; i++) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_first[i], 4);  // one arrival for each warp
            mbar_init(&bar.p_full[i], 4);
            mbar_init(&bar.o_full[i], 1);
        }
        mbar_init(&bar.done, 1);
        fence_barrier_init();
        fence_async_smem();
    }
    grid_dependency_wait();
    // Tensor memory is taken after the wait and before the next kernel may start: a CTA that
    // holds some never waits for a kernel whose CTAs still want theirs.
    if (warp == L::kMmaWarp) {
        tmem_alloc(&tmem_slot, L::kTmem);
        tmem_relinquish();
    }

    // heads of one tile side by side (they share keys in L2), later tiles (more keys) of a
    // sequence first
    const int ny = TILING == kHeads ? a.n_heads / 2 : a.n_heads;
    const int head0 = (int)(blockIdx.x % ny) * (TILING == kHeads ? 2 : 1);
    const int kvh = head0 / (a.n_heads / a.n_kv_heads);
    const int* cu_k = a.cu_k ? a.cu_k : a.cu_q;
    auto usable = [&](int i) {
        return a.cu_q[i] >= 0 && a.cu_q[i + 1] >= a.cu_q[i] && a.cu_q[i + 1] <= a.Tq && cu_k[i] >= 0 && cu_k[i + 1] >= cu_k[i] &&
               cu_k[i + 1] <= a.Tk;
    };
    if (warp == L::kCopyWarp) {
        const int unit = n_units - 1 - (int)(blockIdx.x / ny), b = seq_of_unit<W, 1>(a.cu_q, a.B, unit, lane);
        const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], tile = unit - (q0 / W + b);
        const bool any = usable(b) && tile >= 0 && (int64_t)tile * W < q1 - q0;
        if (lane == 0) s_tile = any ? tile : -1, s_q0 = q0, s_q1 = q1, s_k0 = cu_k[b], s_k1 = cu_k[b + 1];
    } else if (blockIdx.x == 0 && warp < L::kCopyWarp) {  // sequences that no CTA can work on
        for (int i = threadIdx.x; i < a.B; i += 32 * L::kCopyWarp)
            if (!usable(i)) flag_error(a.err, kErrBadContext);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dependents_launch();
    const uint32_t tmem = tmem_slot;
    const int tile = s_tile, q0 = s_q0, q1 = s_q1, k0 = s_k0, k1 = s_k1;
    if (tile < 0) {  // nothing of a sequence
        if (warp == L::kMmaWarp) tmem_dealloc(tmem, L::kTmem);
        return;
    }
    const int off = (k1 - k0) - (q1 - q0);                // query r sees keys 0 .. r + off
    auto head = [&](int i) { return head0 + (TILING == kHeads ? i : 0); };
    auto row0 = [&](int i) { return tile * W + (TILING == kRows ? i * kTile : 0); };
    auto blocks_of = [&](int i) {
        const int rows = min(kTile, q1 - q0 - row0(i));
        const int keys = rows > 0 ? max(0, row0(i) + rows + off) : 0;  // all that the tile's last row sees
        return (keys + kTile - 1) / kTile;
    };
    const int blocks0 = blocks_of(0), blocks1 = TILES == 2 ? blocks_of(1) : 0;
    const int n_blocks = max(blocks0, blocks1);

    auto t_s = [&](int i) { return tmem + 128 * i; };
    auto t_o = [&](int i) { return tmem + TILES * kTile + HD * i; };

    if (warp > L::kMmaWarp) {
        fewer_registers<kRegsOther>();
    } else if (warp == L::kCopyWarp) {
        if constexpr (TILES == 2) fewer_registers<kRegsOther>();
        if (lane == 0 && n_blocks > 0) {
            mbar_arrive_expect_tx(&bar.q_full, TILES * BOXES * kBox);
            for (int i = 0; i < TILES; i++)
                for (int x = 0; x < BOXES; x++)  // an absent second tile reads rows of others, unused
                    tma_load(sq + (i * BOXES + x) * kBox, &map_q, 64 * x, head(i), q0 + row0(i), &bar.q_full);
            int k_sent = 0, v_sent = 0;
            for (int j = 0; j < n_blocks; j++) {
                const int s = j % kStages;
                const uint32_t parity = (j / kStages - 1) & 1;
                if (j >= kStages && !wait_bar(&bar.k_empty[s], parity, a.err)) break;
                mbar_arrive_expect_tx(&bar.k_full[s], BOXES * kBox);
                for (int x = 0; x < BOXES; x++)
                    tma_load(sk + (s * BOXES + x) * kBox, &map_k, 64 * x, kvh, k0 + j * kTile, &bar.k_full[s]);
                k_sent = j + 1;
                if (j >= kStages && !wait_bar(&bar.v_empty[s], parity, a.err)) break;
                mbar_arrive_expect_tx(&bar.v_full[s], BOXES * kBox);
                for (int x = 0; x < BOXES; x++)
                    tma_load(sv + (s * BOXES + x) * kBox, &map_v, 64 * x, kvh, k0 + j * kTile, &bar.v_full[s]);
                v_sent = j + 1;
            }
            // no copy outlives the CTA, also when a wait gave up
            wait_bar(&bar.q_full, 0, a.err);
            for (int j = max(0, k_sent - kStages); j < k_sent; j++) wait_bar(&bar.k_full[j % kStages], (j / kStages) & 1, a.err);
            for (int j = max(0, v_sent - kStages); j < v_sent; j++) wait_bar(&bar.v_full[j % kStages], (j / kStages) & 1, a.err);
        }
    } else if (warp == L::kMmaWarp) {
        if constexpr (TILES == 2) fewer_registers<kRegsOther>();
        const uint64_t dq = desc_sw128(smem_addr(sq), 16), dk = desc_sw128(smem_addr(sk), 16);
        const uint64_t dv = desc_sw128(smem_addr(sv), kBox);
        constexpr uint64_t kBlock = BOXES * kBox >> 4;    // one operand block, in descriptor units
        auto issue_s = [&](int i, int j) {                // S_i = Q_i K(j)^T
            const uint64_t q = dq + i * kBlock, k = dk + (j % kStages) * kBlock;
#pragma unroll
            for (int x = 0; x < HD / 16; x++) {           // 16 dims = 32 bytes, 4 of them to a box
                const uint32_t at = (x / 4) * (kBox >> 4) + (x % 4) * 2;
                umma_bf16(t_s(i), q + at, k + at, idesc16<T>(kTile, false), x > 0);
            }
            umma_commit(&bar.s_full[i]);
            // the last of the block's readers frees it
            if (i == 1 || j >= blocks1) umma_commit(&bar.k_empty[j % kStages]);
        };
        auto issue_o = [&](int i, int j, int steps, auto from, auto to) {  // O_i += P_i V(j) of keys from .. to - 1
            const uint64_t v = dv + (j % kStages) * kBlock;
#pragma unroll
            for (int k = decltype(from)::value / 16; k < decltype(to)::value / 16; k++)  // 16 keys: 8 columns of P, 2048 bytes of values
                if (k < steps) umma_tmem_a(t_o(i), t_s(i) + 8 * k, v + k * (2048 >> 4), idesc16<T>(HD, true), j > 0 || k > 0);
        };
        using Zero = std::integral_constant<int, 0>;
        using First = std::integral_constant<int, kFirst>;
        using All = std::integral_constant<int, kTile>;
        // V(j), with the rows behind the last key set to zero up to a multiple of 16
        auto values_ready = [&](int j) {
            if (!wait_bar(&bar.v_full[j % kStages], (j / kStages) & 1, a.err)) return false;
            const int left = k1 - k0 - j * kTile, pad = (16 - left % 16) % 16;
            if (left < kTile && pad) {
                for (int e = lane; e < pad * 8 * BOXES; e += 32)
                    *reinterpret_cast<uint4*>(sv + ((j % kStages) * BOXES + e / (8 * pad)) * kBox + left * 128 + e % (8 * pad) * 16) =
                        make_uint4(0, 0, 0, 0);
                fence_async_smem();
                __syncwarp();
            }
            return true;
        };
        bool ok = n_blocks > 0 && wait_bar(&bar.q_full, 0, a.err) && wait_bar(&bar.k_full[0], 0, a.err);
        if (ok && elect_one()) {
            if (blocks0 > 0) issue_s(0, 0);
            if (blocks1 > 0) issue_s(1, 0);
        }
        // All copies of an iteration are waited for at its start, while the last S is still being
        // computed: an issue blocks until the tensor cores take it, and what stands between two
        // issues lets them run dry.
        for (int j = 0; j < n_blocks && ok; j++) {
            const int steps = (min(k1 - k0 - j * kTile, kTile) + 15) / 16;
            ok = values_ready(j) && (j + 1 >= n_blocks || wait_bar(&bar.k_full[(j + 1) % kStages], ((j + 1) / kStages) & 1, a.err));
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                const int blocks = i ? blocks1 : blocks0;
                if (!ok || j >= blocks) continue;
                ok = wait_bar(&bar.p_first[i], j & 1, a.err);
                if (!ok) continue;
                tc_fence_after();
                if (elect_one()) issue_o(i, j, steps, Zero(), First());
                ok = wait_bar(&bar.p_full[i], j & 1, a.err);
                if (!ok) continue;
                tc_fence_after();
                if (elect_one()) {
                    issue_o(i, j, steps, First(), All());
                    if (i == 1 || j >= blocks1) umma_commit(&bar.v_empty[j % kStages]);
                    if (j + 1 < blocks) issue_s(i, j + 1);
                    else umma_commit(&bar.o_full[i]);
                }
            }
        }
        if (!ok && n_blocks > 0) {  // a wait gave up: let the products in flight end
            if (elect_one()) umma_commit(&bar.done);
            wait_bar(&bar.done, 0, a.err);
        }
        __syncwarp();
    } else {
        if constexpr (TILES == 2) more_registers<kRegsSoftmax>();
        const int i = warp >> 2;                          // tile
        const int blocks = i ? blocks1 : blocks0, first = row0(i);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
        const uint32_t ts = t_s(i) + lanes, to = t_o(i) + lanes;
        const int r = first + (warp & 3) * 32 + lane;   // row within the sequence
        const float scale = kLog2e * rsqrtf((float)HD);
        const unsigned long long scale2 = pack2(__float_as_uint(scale), __float_as_uint(scale));
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < blocks; j++) {
            ok = __all_sync(0xffffffffu, wait_bar(&bar.s_full[i], j & 1, a.err));
            if (!ok) break;
            tc_fence_after();
            const int limit = r + off - j * kTile;        // last column this row sees
            const bool edge = j * kTile + kTile - 1 > first + off;
            uint32_t v[kTile];
#pragma unroll
            for (int c = 0; c < kTile; c += 32) tmem_ld32_async(ts + c, v + c);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < kTile; c += 32) tmem_regs_ready(v + c);
            if (edge) mask_row<kTile>(v, limit);
            // The first half's weights are taken from the maximum so far while the block's is being
            // found, and once more in the rare block that moves it (and in the first one).
            unsigned long long shift2, sum[2];
            bool moved = false;
            while (true) {
                const float shift = m == -INFINITY ? 0.0f : -m;
                shift2 = pack2(__float_as_uint(shift), __float_as_uint(shift));
                sum[0] = sum[1] = 0;
                weights<T, kFirst>(v, scale2, shift2, sum, ts);
                if (moved) break;
                const float top = max_row<kTile>(v) * scale;
                const bool grows = top > m + kLazy;
                if (!__any_sync(0xffffffffu, grows)) break;
                const float corr = !grows ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - top);
                if (grows) m = top;
                l *= corr;
                if (j > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        uint32_t w[16];
                        tmem_ld16(to + c, o);
#pragma unroll
                        for (int k = 0; k < 16; k++) w[k] = __float_as_uint(o[k] * corr);
                        tmem_st16(to + c, w);
                    }
                }
                // stores to the same columns are not ordered among themselves: the old maximum's
                // weights have to be there before the new one's go over them
                tmem_wait_st();
                moved = true;
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.p_first[i]);
            weights<T, kTile - kFirst>(v + kFirst, scale2, shift2, sum, ts + kFirst / 2);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.p_full[i]);
            uint32_t a0, a1;
            unpack2(add2(sum[0], sum[1]), a0, a1);
            l += __uint_as_float(a0) + __uint_as_float(a1);
        }
        if (ok && blocks > 0) {
            ok = __all_sync(0xffffffffu, wait_bar(&bar.o_full[i], 0, a.err));
            tc_fence_after();
        }
        if (ok && first < q1 - q0) {
            const bool none = r + off < 0;                // saw no key: zeros, whatever O holds
            const float inv = 1.0f / l;
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
                    for (int e = 0; e < 4; e++)
                        w[e] = none ? 0u : pack16<T>(__uint_as_float(o[k + 2 * e]) * inv, __uint_as_float(o[k + 2 * e + 1]) * inv);
                    *reinterpret_cast<uint4*>(out + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == L::kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, L::kTmem);
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

template <typename T, int HD, Tiling TILING>
cudaError_t launch_tiles(const PromptAttnArgs& a, cudaStream_t s) {
    using L = Layout<HD, TILING>;
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is set
    int dev = 0;
    cudaError_t rc = cudaGetDevice(&dev);
    if (rc != cudaSuccess) return rc;
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        rc = cudaFuncSetAttribute(prompt_attn_kernel<T, HD, TILING>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
        if (rc != cudaSuccess) return rc;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev);
    }
    if (!encode_fn()) return cudaErrorNotSupported;
    CUtensorMap mq, mk, mv;
    if (!encode(&mq, a.dtype, a.q, a.q_stride, a.Tq, a.n_heads, HD) ||
        !encode(&mk, a.dtype, a.k, a.k_stride, a.Tk, a.n_kv_heads, HD) ||
        !encode(&mv, a.dtype, a.v, a.v_stride, a.Tk, a.n_kv_heads, HD))
        return cudaErrorInvalidValue;
    const int units = a.Tq / L::kRowsPerUnit + a.B;
    const int64_t grid = (int64_t)units * (TILING == kHeads ? a.n_heads / 2 : a.n_heads);
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    count_launch();
    return launch_ex(prompt_attn_kernel<T, HD, TILING>, dim3((unsigned)grid), dim3(L::kThreads), L::kSmem, s, 1, mq, mk, mv, a, units);
}

template <typename T>
cudaError_t launch_t(const PromptAttnArgs& a, cudaStream_t s) {
    if (a.head_dim == 64) return launch_tiles<T, 64, kOne>(a, s);
    // Prompts of 32 keys and less on average: a CTA lives a few microseconds and waits most of
    // them, so two smaller ones to an SM, each with one block of rows (32 prompts of 7 tokens, 21
    // heads: 27.8 -> 17.3 us; 64 of 40, 32 heads: 58.5 -> 56.5; but 8 of 64: 9.5 -> 11.9).  The
    // average is what the host knows: a long prompt among many of one token pays for it (63 of
    // one and one of 1900, 32 heads: 81 us, the long one alone 35).
    if (a.Tk / a.B <= 32) return launch_tiles<T, 128, kOne>(a, s);
    return a.n_heads / a.n_kv_heads % 2 ? launch_tiles<T, 128, kRows>(a, s) : launch_tiles<T, 128, kHeads>(a, s);
}

}  // namespace

cudaError_t launch_prompt_attention(const PromptAttnArgs& a, cudaStream_t s) {
    return a.dtype == kBF16 ? launch_t<__nv_bfloat16>(a, s) : launch_t<__half>(a, s);
}

}  // namespace nitro
