// Token log probabilities, entropy and top alternatives (nr_token_logprobs).
//
// One read of the logits.  A cluster of 1 to 8 CTAs takes a row, each CTA a run of its
// 16-byte vectors, each thread every 256th of them: running reference m (moved only when a
// vector's maximum passes it by 8), sum S of e^(x - m) and W of e^(x - m) (x - m), from which
//
//   log p(x) = (x - m) - log S,   entropy = log S - W / S.
//
// x - m is taken before the factor log2 e, so that large logits keep their differences.
//
// Top k without a second pass: every thread also keeps its largest vector maximum.  With the
// keys (value, vector number) ordered by larger value, then smaller number, let K be the k-th
// largest thread key.  k elements are as large as K or larger, so every element of the top k
// is, and such elements are found in those k threads' vectors alone: only these (1/8 of the
// row at k = 32) are looked at again, while they are in L2.  The few candidates are ranked by
// counting the larger ones (ids make all keys distinct, so equal logits fall in order of their
// ids), the lists of a cluster's CTAs are joined the same way through distributed shared
// memory.  Rows that hold a NaN or +inf and more candidates than the buffer holds take k
// passes instead.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cmath>

#include "kv8.h"
#include "kernels.h"
#include "packed_rows.cuh"

namespace nitro {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;       // NR_LOGPROBS_MAX_TOP
constexpr int kCandidates = 1024;
constexpr int kMaxCluster = 8;
constexpr int kBatch = 4;         // vectors in flight for each thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;
constexpr float kNothing = -1e4f; // e^-10^4 is 0, and 0 * -10^4 too

using Key = unsigned long long;

// Orders (value, number): larger value first, then smaller number; NaN below -inf; +0 and -0
// are one value.  Never 0 for a number below 2^31.
__device__ __forceinline__ Key rank_key(float v, int n) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    const uint32_t o = v != v ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((Key)o << 32) | (0xffffffffu - (uint32_t)n);
}
__device__ __forceinline__ int key_number(Key k) { return (int)(0xffffffffu - (uint32_t)k); }
// The value of a key that is not a NaN's.
__device__ __forceinline__ float key_value(Key k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A row as 16-byte aligned vectors; the first and last may reach over its ends.
template <typename T>
struct RowView {
    static constexpr int N = 16 / (int)sizeof(T);
    const T* p;   // element 0
    int lead;     // elements of vector 0 before it
    int V;
    __device__ __forceinline__ RowView(const T* row, int v) : p(row), lead((int)((uintptr_t)row % 16 / sizeof(T))), V(v) {}
    __device__ __forceinline__ int vectors() const { return (int)(((int64_t)V + lead + N - 1) / N); }
    // id of vector i's first element (negative, if it is before the row)
    __device__ __forceinline__ int64_t base(int i) const { return (int64_t)i * N - lead; }
    // elements of vector i, what lies outside the row as -inf
    __device__ __forceinline__ uint4 load(int i) const {
        const int64_t b = base(i);
        if (b >= 0 && b + N <= V) {
            uint4 u;
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p + b));
            return u;
        }
        uint4 u;
        T* t = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int k = 0; k < N; k++) t[k] = b + k >= 0 && b + k < V ? p[b + k] : from_f32<T>(-INFINITY);
        return u;
    }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float* x) {
    const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int k = 0; k < RowView<T>::N; k++) x[k] = to_f32(t[k]);
}

struct Stats {
    float m, s, w;  // reference (-inf: nothing but -inf seen), sum, weighted sum
};

// The same sums under the reference `to` (to >= m).
__device__ __forceinline__ Stats moved(Stats a, float to) {
    if (a.m == to) return a;
    if (a.m == -INFINITY) return {to, a.s, a.w};  // zeros, or a bad part's NaN
    const float d = a.m - to, f = exp2_fast(d * kLog2e);
    return {to, a.s * f, f == 0.0f ? 0.0f : (a.w + a.s * d) * f};
}
__device__ __forceinline__ Stats join(Stats a, Stats b) {
    const float m = fmaxf(a.m, b.m);
    a = moved(a, m);
    b = moved(b, m);
    return {m, a.s + b.s, a.w + b.w};
}

// One vector of N values into a thread's running sums.
template <int N>
__device__ __forceinline__ void take(const float* x, float top, Stats& a) {
    if (top > a.m + kLazy) a = moved(a, top);
    const float m = a.m == -INFINITY ? 0.0f : a.m;
    const unsigned long long m2 = pack2(__float_as_uint(m), __float_as_uint(m));
    const unsigned long long log2e = pack2(__float_as_uint(kLog2e), __float_as_uint(kLog2e));
    unsigned long long s = 0, w = 0;
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        uint32_t d0, d1, y0, y1;
        unpack2(sub2(pack2(__float_as_uint(x[k]), __float_as_uint(x[k + 1])), m2), d0, d1);
        const unsigned long long d = pack2(__float_as_uint(fmaxf(__uint_as_float(d0), kNothing)),
                                           __float_as_uint(fmaxf(__uint_as_float(d1), kNothing)));
        unpack2(mul2(d, log2e), y0, y1);
        const unsigned long long e = pack2(__float_as_uint(exp2_fast(__uint_as_float(y0))),
                                           __float_as_uint(exp2_fast(__uint_as_float(y1))));
        s = k ? add2(s, e) : e;
        w = fma2(e, d, w);
    }
    uint32_t s0, s1, w0, w1;
    unpack2(s, s0, s1);
    unpack2(w, w0, w1);
    a.s += __uint_as_float(s0) + __uint_as_float(s1);
    a.w += __uint_as_float(w0) + __uint_as_float(w1);
}

struct Shared {
    Stats stats[kThreads / 32];
    Stats all;             // of the CTA
    int bad;               // a NaN in the CTA's part
    int count;             // candidates
    int chosen[kMaxTop];   // threads whose vectors are looked at again
    Key bound;
    Key top[kMaxTop];      // the CTA's list
    union {
        Key keys[kCandidates];
        Key thread_key[kThreads];
    };
};

// Ranks the n distinct keys and writes the first k of them in order.
__device__ __forceinline__ void rank_keys(const Key* keys, int n, int k, Key* out) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const Key mine = keys[i];
        int larger = 0;
        for (int j = 0; j < n; j++) larger += keys[j] > mine;
        if (larger < k) out[larger] = mine;
    }
}

// The k largest keys of vectors v0 .. v1 - 1, one pass for each.
template <typename T>
__device__ void top_by_passes(const RowView<T>& row, int v0, int v1, int k, Shared& sh) {
    Key last = ~0ull;
    for (int r = 0; r < k; r++) {
        Key best = 0;
        for (int v = v0 + threadIdx.x; v < v1; v += kThreads) {
            float x[RowView<T>::N];
            unpack<T>(row.load(v), x);
#pragma unroll
            for (int e = 0; e < RowView<T>::N; e++) {
                const int64_t id = row.base(v) + e;
                if (id < 0 || id >= row.V) continue;
                const Key key = rank_key(x[e], (int)id);
                if (key < last && key > best) best = key;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Key q = __shfl_xor_sync(0xffffffffu, best, o);
            best = q > best ? q : best;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.keys[threadIdx.x >> 5] = best;
        __syncthreads();
        best = sh.keys[0];
        for (int i = 1; i < kThreads / 32; i++) best = sh.keys[i] > best ? sh.keys[i] : best;
        last = best;
        if (threadIdx.x == 0) sh.top[r] = best;  // 0: the part has fewer elements
        if (best == 0) last = 0;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_kernel(LogprobArgs a, int cluster) {
    constexpr int N = RowView<T>::N;
    __shared__ Shared sh;
    __shared__ Key lists[kMaxCluster * kMaxTop];
    const int t = threadIdx.x, lane = t & 31, rank = blockIdx.x % cluster;
    const int64_t m_row = blockIdx.x / cluster;
    grid_dependency_wait();
    grid_dependents_launch();
    const RowView<T> row((const T*)a.logits + m_row * a.row_stride, a.V);
    const int nv = row.vectors(), per = (nv + cluster - 1) / cluster;
    const int v0 = min(rank * per, nv), v1 = min(nv, v0 + per);

    // the pass over this CTA's vectors
    Stats st{-INFINITY, 0.0f, 0.0f};
    float best = -INFINITY;
    int best_v = v0 + t;
    bool nan = false;
    auto fetch = [&](uint4* u, int v) {
#pragma unroll
        for (int i = 0; i < kBatch; i++)
            if (v + i * kThreads < v1) u[i] = row.load(v + i * kThreads);
    };
    auto use = [&](const uint4* u, int v) {
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            if (v + i * kThreads >= v1) break;
            float x[N];
            unpack<T>(u[i], x);
            float top = x[0];
#pragma unroll
            for (int k = 1; k < N; k++) top = max_nan(top, x[k]);
            nan |= top != top;
            if (top > best) best = top, best_v = v + i * kThreads;
            take<N>(x, top, st);
        }
    };
    {
        uint4 u[2][kBatch];
        const int step = kBatch * kThreads;
        fetch(u[0], v0 + t);
        for (int v = v0 + t; v < v1; v += 2 * step) {
            fetch(u[1], v + step);
            use(u[0], v);
            fetch(u[0], v + 2 * step);
            use(u[1], v + step);
        }
    }

    // the CTA's sums
    Stats sum = st;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stats q{__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o),
                      __shfl_xor_sync(0xffffffffu, sum.w, o)};
        sum = join(sum, q);
    }
    const int k = a.top_k;
    if (lane == 0) sh.stats[t >> 5] = sum;
    if (t == 0) sh.count = 0, sh.bound = 0;
    if (k) sh.thread_key[t] = v0 + t < v1 ? rank_key(best, best_v) : 0;
    const bool bad = __syncthreads_or(nan);
    if (t < 32) {
        sum = lane < kThreads / 32 ? sh.stats[lane] : Stats{-INFINITY, 0.0f, 0.0f};
#pragma unroll
        for (int o = kThreads / 64; o > 0; o >>= 1) {
            const Stats q{__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o),
                          __shfl_xor_sync(0xffffffffu, sum.w, o)};
            sum = join(sum, q);
        }
        if (lane == 0) {
            if (bad || sum.m == INFINITY) sum.s = NAN;  // no statistics of such a row
            sh.all = sum;
            sh.bad = bad;
        }
    }

    // the CTA's top k
    if (k) {
        const Key mine = sh.thread_key[t];
        int larger = 0;
#pragma unroll 8
        for (int j = 0; j < kThreads; j += 2) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(&sh.thread_key[j]);
            larger += (q.x > mine) + (q.y > mine);
        }
        if (mine && larger < k) sh.chosen[larger] = t;
        if (larger == k - 1 && mine) sh.bound = mine;  // stays 0 where fewer than k threads have vectors
        const int chosen = min(k, min(kThreads, v1 - v0));
        __syncthreads();
        if (!bad) {
            const Key bound = sh.bound;
            for (int c = t >> 5; c < chosen; c += kThreads / 32)
                for (int v = v0 + sh.chosen[c] + lane * kThreads; v < v1; v += 32 * kThreads) {
                    float x[N];
                    unpack<T>(row.load(v), x);
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const int64_t id = row.base(v) + e;
                        if (id < 0 || id >= a.V || rank_key(x[e], v) < bound) continue;
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < kCandidates) sh.keys[at] = rank_key(x[e], (int)id);
                    }
                }
        }
        __syncthreads();
        if (t < k) sh.top[t] = 0;
        __syncthreads();
        if (bad || sh.count > kCandidates) top_by_passes(row, v0, v1, k, sh);
        else rank_keys(sh.keys, sh.count, k, sh.top);
    }

    // the cluster's
    Stats all;
    const Key* list = sh.top;
    if (cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (rank == 0) {
            all = sh.all;
            for (int r = 1; r < cluster; r++) all = join(all, cl.map_shared_rank(&sh, r)->all);
            for (int i = t; i < cluster * k; i += kThreads) lists[i] = cl.map_shared_rank(&sh, i / k)->top[i % k];
        }
        cl.sync();  // no CTA leaves while its list is read
        if (rank) return;
        if (k) {
            // absent entries are 0: they rank behind every key, in any order
            for (int i = t; i < cluster * k; i += kThreads) {
                const Key mine = lists[i];
                int larger = 0;
                for (int j = 0; j < cluster * k; j++) larger += lists[j] > mine;
                if (mine && larger < k) sh.top[larger] = mine;
            }
        }
    } else {
        __syncthreads();
        all = sh.all;
    }
    __syncthreads();
    const float ls = all.s > 0.0f || all.s != all.s ? logf(all.s) : NAN;
    if (t == 0) {
        if (a.targets) {
            const int id = a.targets[m_row];
            a.target_logprob[m_row] = id < 0 || id >= a.V ? NAN : (to_f32(row.p[id]) - all.m) - ls;
        }
        if (a.entropy) a.entropy[m_row] = ls - all.w / all.s;
    }
    if (t < k) {
        const Key key = list[t];
        a.top_ids[m_row * k + t] = key_number(key);
        a.top_logprob[m_row * k + t] = (key_value(key) - all.m) - ls;
    }
}

template <typename T>
cudaError_t launch_t(const LogprobArgs& a, cudaStream_t s) {
    // More CTAs to a row while it has over 4096 elements for each and they all fit the device at
    // once: few rows are bound by latency, many by memory, where a CTA for each row has the
    // least to join.
    int cluster = 1;
    while (cluster < kMaxCluster && a.V / cluster > 4096 && (int64_t)a.M * cluster * 2 <= 148 * 4) cluster *= 2;
    count_launch();
    return launch_ex(logprob_kernel<T>, dim3((unsigned)((int64_t)a.M * cluster)), dim3(kThreads), 0, s, (unsigned)cluster, a, cluster);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, cudaStream_t s) {
    if (a.dtype == kF32) return launch_t<float>(a, s);
    return a.dtype == kBF16 ? launch_t<__nv_bfloat16>(a, s) : launch_t<__half>(a, s);
}

}  // namespace nitro
