// Token log probabilities, entropy and top alternatives (nr_token_logprobs).
//
// One read of the logits.  A cluster of 1 to 8 CTAs takes a row, each CTA a run of its
// 32-byte vectors, each thread every 256th of them: running reference m (moved only when a
// vector's maximum passes it by 8), sum S of e^(x - m) and W of e^(x - m) (x - m), from which
//
//   log p(x) = (x - m) - log S,   entropy = log S - W / S.
//
// x - m is taken before the factor log2 e, so that large logits keep their differences.
//
// Top k without a second pass: every thread also keeps its largest vector maximum.  With the
// keys (value, vector number) ordered by larger value, then smaller number, let K be the
// smallest, over the CTA's w full warps, of a warp's ceil(k/w)-th largest thread key.  Then k
// elements at least are as large as K or larger, so every element of the top k is, and such
// elements are found only in vectors of the few threads whose key is: the thread's two best
// ones, and all of them if its third largest maximum is as large as K, are looked at again
// while they are in L2.  The candidates are ranked by counting the larger ones (ids
// make all keys distinct, so equal logits fall in order of their ids), the lists of a
// cluster's CTAs are joined the same way through distributed shared memory.  Rows that hold a
// NaN and more candidates than the buffer holds take k passes instead.
//
// Measured: 2048 rows of 128256 bf16 logits, top 20: 111 us, 4.74 TB/s, 0.72 of the measured copy
// bandwidth (98 us without a top list; 1024 rows of fp32 logits 5.5 TB/s, 0.84, without a list 6.0, 0.92): two elements of 16 bits
// for each of 32 need twice the exponentials (8 cycles a warp) and sums for the same bytes,
// and the candidates' latency is hidden only by the SM's other rows.  64 rows of 32000 fp32:
// 9.2 us, a chain of latencies.  A ninth warp that finishes a row while the others stream
// the next one was slower (140 us: fewer registers and a longer chain on one warp).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

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

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ __half low_of(__half2 v) { return __low2half(v); }
__device__ __forceinline__ __half high_of(__half2 v) { return __high2half(v); }
__device__ __forceinline__ __nv_bfloat16 low_of(__nv_bfloat162 v) { return __low2bfloat16(v); }
__device__ __forceinline__ __nv_bfloat16 high_of(__nv_bfloat162 v) { return __high2bfloat16(v); }

// A row as 32-byte aligned vectors; the first and last may reach over its ends.
template <typename T>
struct RowView {
    static constexpr int N = 32 / (int)sizeof(T);
    struct Vec {
        uint32_t u[8];
    };
    const T* p;   // element 0
    int lead;     // elements of vector 0 before it
    int V;
    __device__ __forceinline__ RowView(const T* row, int v) : p(row), lead((int)((uintptr_t)row % 32 / sizeof(T))), V(v) {}
    __device__ __forceinline__ int vectors() const { return (int)(((int64_t)V + lead + N - 1) / N); }
    // id of vector i's first element (negative, if it is before the row)
    __device__ __forceinline__ int64_t base(int i) const { return (int64_t)i * N - lead; }
    // vectors that lie inside the row
    __device__ __forceinline__ int first_whole() const { return lead ? 1 : 0; }
    __device__ __forceinline__ int end_whole() const { return (int)(((int64_t)V + lead) / N); }
    __device__ __forceinline__ Vec load_whole(int i) const { return load_whole_at(p + base(i)); }
    static __device__ __forceinline__ Vec load_whole_at(const T* at) {
        Vec v;
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(v.u[0]), "=r"(v.u[1]), "=r"(v.u[2]), "=r"(v.u[3]), "=r"(v.u[4]), "=r"(v.u[5]), "=r"(v.u[6]), "=r"(v.u[7])
                     : "l"(at));
        return v;
    }
    // elements of any vector i, what lies outside the row as -inf
    __device__ __noinline__ Vec load(int i) const {
        const int64_t b = base(i);
        Vec v;
        T t[N];
#pragma unroll
        for (int k = 0; k < N; k++) t[k] = b + k >= 0 && b + k < V ? p[b + k] : from_f32<T>(-INFINITY);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if constexpr (sizeof(T) == 4) {
                v.u[k] = __float_as_uint(to_f32(t[k]));
            } else {
                uint16_t h[2];
                memcpy(h, &t[2 * k], 4);
                v.u[k] = h[0] | (uint32_t)h[1] << 16;
            }
        }
        return v;
    }
};

template <typename T>
__device__ __forceinline__ void unpack(const typename RowView<T>::Vec& v, float* x) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if constexpr (std::is_same<T, float>::value) {
            x[k] = __uint_as_float(v.u[k]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            x[2 * k] = __uint_as_float(v.u[k] << 16);
            x[2 * k + 1] = __uint_as_float(v.u[k] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v.u[k]));
            x[2 * k] = f.x;
            x[2 * k + 1] = f.y;
        }
    }
}

// The largest element, NaN if there is one.
template <typename T>
__device__ __forceinline__ float vec_max(const typename RowView<T>::Vec& v) {
    if constexpr (std::is_same<T, float>::value) {
        float t = __uint_as_float(v.u[0]);
#pragma unroll
        for (int k = 1; k < 8; k++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(t) : "f"(__uint_as_float(v.u[k])));
        return t;
    } else {
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        T2 t[8];
#pragma unroll
        for (int k = 0; k < 8; k++) t[k] = *reinterpret_cast<const T2*>(&v.u[k]);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < o; k++) t[k] = __hmax2_nan(t[k], t[k + o]);
        return to_f32(__hmax_nan(low_of(t[0]), high_of(t[0])));
    }
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

// x - m of one element; the 16-bit types' subtraction widens its operand itself.
__device__ __forceinline__ float less(uint32_t x, float m, float) { return __uint_as_float(x) - m; }
__device__ __forceinline__ float less(uint16_t x, float m, __nv_bfloat16) {
    float d;
    asm("sub.rn.f32.bf16 %0, %1, %2;" : "=f"(d) : "h"(x), "f"(m));
    return d;
}
__device__ __forceinline__ float less(uint16_t x, float m, __half) {
    float d;
    asm("sub.rn.f32.f16 %0, %1, %2;" : "=f"(d) : "h"(x), "f"(m));
    return d;
}

// Sums of one vector.  e^-inf * -inf is NaN: with CLAMP such values count as nothing, without
// it the weighted sum tells that there is one.
template <typename T, bool CLAMP>
__device__ __forceinline__ void sums_of(const typename RowView<T>::Vec& v, float m, float& s, float& w) {
    if constexpr (sizeof(T) == 2 && !CLAMP) {
        // bound by issue slots: two elements to a product or sum (115 -> 111 us for 2048 rows of
        // 128256; the other forms, bound by memory or rare, gain nothing: 9.2 -> 9.3 us for 64 rows
        // of 32000 fp32)
        const unsigned long long log2e = pack2(__float_as_uint(kLog2e), __float_as_uint(kLog2e));
        unsigned long long s2 = 0, w2 = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float d0 = less((uint16_t)v.u[k], m, T()), d1 = less((uint16_t)(v.u[k] >> 16), m, T());
            const unsigned long long d = pack2(__float_as_uint(d0), __float_as_uint(d1));
            uint32_t y0, y1;
            unpack2(mul2(d, log2e), y0, y1);
            const unsigned long long e = pack2(__float_as_uint(exp2_fast(__uint_as_float(y0))), __float_as_uint(exp2_fast(__uint_as_float(y1))));
            s2 = add2(s2, e);
            w2 = fma2(e, d, w2);
        }
        uint32_t lo, hi;
        unpack2(s2, lo, hi);
        s = __uint_as_float(lo) + __uint_as_float(hi);
        unpack2(w2, lo, hi);
        w = __uint_as_float(lo) + __uint_as_float(hi);
        return;
    }
    float ss[2] = {0.0f, 0.0f}, ww[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < RowView<T>::N; k++) {
        float d;
        if constexpr (sizeof(T) == 4) d = less(v.u[k], m, T());
        else d = less((uint16_t)(v.u[k / 2] >> (16 * (k & 1))), m, T());
        if (CLAMP) d = fmaxf(d, kNothing);
        const float e = exp2_fast(d * kLog2e);
        ss[k & 1] += e;
        ww[k & 1] = fmaf(e, d, ww[k & 1]);
    }
    s = ss[0] + ss[1];
    w = ww[0] + ww[1];
}

// One vector into a thread's running sums; `masked`: whether it has met a -inf, `nan` a NaN.
template <typename T>
__device__ __forceinline__ void take(const typename RowView<T>::Vec& v, float top, Stats& a, bool& masked, bool& nan) {
    if (top > a.m + kLazy) a = moved(a, top);
    const float m = a.m == -INFINITY ? 0.0f : a.m;
    float s, w;
    if (!masked) {
        sums_of<T, false>(v, m, s, w);
        masked = w != w;
    }
    if (masked) {
        nan |= top != top;
        sums_of<T, true>(v, m, s, w);
    }
    a.s += s;
    a.w += w;
}

struct Shared {
    Stats stats[kThreads / 32];
    Stats all;             // of the CTA
    int bad;               // a NaN in the CTA's part
    int count;             // candidates
    int n_chosen;
    int chosen[kThreads];  // threads whose vectors are looked at again
    Key warp_key[kThreads / 32];
    Key top[kMaxTop];      // the CTA's list
    Key keys[kCandidates];
};

// Largest key of the warp.
__device__ __forceinline__ Key warp_max_key(Key k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((Key)hi << 32) | lo;
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
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 4 : 5) logprob_kernel(LogprobArgs a, int cluster) {
    constexpr int N = RowView<T>::N;
    __shared__ Shared sh;
    const int t = threadIdx.x, lane = t & 31, rank = blockIdx.x % cluster;
    const int64_t m_row = blockIdx.x / cluster;
    grid_dependency_wait();
    grid_dependents_launch();
    const RowView<T> row((const T*)a.logits + m_row * a.row_stride, a.V);
    const int nv = row.vectors(), per = (nv + cluster - 1) / cluster;
    const int v0 = min(rank * per, nv), v1 = min(nv, v0 + per);

    if (t < kMaxTop) sh.top[t] = 0;
    if (t == 0) sh.count = sh.n_chosen = 0;

    // the pass over this CTA's vectors
    Stats st{-INFINITY, 0.0f, 0.0f};
    float best = -INFINITY, second = -INFINITY, third = -INFINITY;
    int best_v = v0 + t, second_v = -1;
    bool nan = false, masked = false;
    using Vec = typename RowView<T>::Vec;
    const int w0 = row.first_whole(), w1 = min(v1, row.end_whole());
    auto use = [&](const Vec& u, int v) {
        const float top = vec_max<T>(u);
        third = fmaxf(third, fminf(top, second));
        if (top > best) second = best, second_v = best_v, best = top, best_v = v;
        else if (top > second) second = top, second_v = v;
        take<T>(u, top, st, masked, nan);
    };
    {
        // a thread's first and last vector may reach over the row's ends, the others are whole
        int v = v0 + t;
        if (v < v1 && v < w0) use(row.load(v), v), v += kThreads;
        const int n = w1 > v ? (w1 - v + kThreads - 1) / kThreads : 0;
        const T* p = row.p + row.base(v);
        auto whole = [&](int i) { return row.load_whole_at(p + (int64_t)i * (kThreads * N)); };
        Vec a, b;
        if (n > 0) a = whole(0);
        if (n > 1) b = whole(1);
        int i = 0;
        for (; i + 3 < n; i += 2) {
            use(a, v + i * kThreads);
            a = whole(i + 2);
            use(b, v + (i + 1) * kThreads);
            b = whole(i + 3);
        }
        if (i < n) use(a, v + i * kThreads);
        if (i + 2 < n) a = whole(i + 2);
        if (i + 1 < n) use(b, v + (i + 1) * kThreads);
        if (i + 2 < n) use(a, v + (i + 2) * kThreads);
        const int edge = nv - 1;
        if (edge >= w1 && edge >= max(v0, w0) && edge < v1 && (edge - v0) % kThreads == t) use(row.load(edge), edge);
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
    const Key mine = k && v0 + t < v1 ? rank_key(best, best_v) : 0;
    const int full = min(kThreads, v1 - v0) / 32;  // warps whose every thread has vectors
    if (k && (t >> 5) < full) {
        Key left = mine, top = 0;
        for (int r = 0; r < (k + full - 1) / full; r++) {
            top = warp_max_key(left);
            if (left == top) left = 0;
        }
        if (lane == 0) sh.warp_key[t >> 5] = top;
    }
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
        Key bound = full ? ~0ull : 0;
        for (int w = 0; w < full; w++) bound = sh.warp_key[w] < bound ? sh.warp_key[w] : bound;
        const float least = bound ? key_value(bound) : -INFINITY;
        auto look = [&](const Vec& u, int v) {
            uint32_t hits = 0;
            float x[N];
            unpack<T>(u, x);
#pragma unroll
            for (int e = 0; e < N; e++) hits |= (x[e] >= least ? 1u : 0u) << e;
            for (; hits; hits &= hits - 1) {
                const int e = __ffs(hits) - 1;
                const int64_t id = row.base(v) + e;
                float value = x[0];
#pragma unroll
                for (int j = 1; j < N; j++) value = e == j ? x[j] : value;
                if (id < 0 || id >= a.V || rank_key(value, v) < bound) continue;
                const int at = atomicAdd(&sh.count, 1);
                if (at < kCandidates) sh.keys[at] = rank_key(value, (int)id);
            }
        };
        auto any = [&](int v) { return v >= w0 && v < w1 ? row.load_whole(v) : row.load(v); };
        if (!full) {  // so few vectors that all their elements are ranked
            const int64_t from = row.base(v0) < 0 ? 0 : row.base(v0);
            const int n = (int)(min((int64_t)a.V, row.base(v1)) - from);
            for (int i = t; i < n; i += kThreads) sh.keys[i] = rank_key(to_f32(row.p[from + i]), (int)(from + i));
            if (t == 0) sh.count = max(n, 0);
        } else if (!bad && mine && mine >= bound) {
            if (third >= least) {
                sh.chosen[atomicAdd(&sh.n_chosen, 1)] = t;
            } else {
                const bool two = second_v >= 0 && second >= least;
                const Vec x = any(best_v), y = any(two ? second_v : best_v);
                look(x, best_v);
                if (two) look(y, second_v);
            }
        }
        __syncthreads();
        const int chosen = sh.n_chosen;
        if (chosen) {
            for (int c = t >> 5; c < chosen; c += kThreads / 32)
                for (int v = v0 + sh.chosen[c] + lane * kThreads; v < v1; v += 32 * kThreads) look(any(v), v);
            __syncthreads();
        }
        if ((bad && full) || sh.count > kCandidates) {
            top_by_passes(row, v0, v1, k, sh);
        } else {
            // four threads to a candidate
            const int n = sh.count;
            for (int i = t / 4; i < (n + 7) / 8 * 8; i += kThreads / 4) {
                const Key key = i < n ? sh.keys[i] : 0;
                int larger = 0;
                for (int j = t % 4; j < n; j += 4) larger += sh.keys[j] > key;
                larger += __shfl_xor_sync(0xffffffffu, larger, 1);
                larger += __shfl_xor_sync(0xffffffffu, larger, 2);
                if (i < n && larger < k && t % 4 == 0) sh.top[larger] = key;
            }
        }
    }

    __syncthreads();
    Stats all = sh.all;
    Key key = t < k ? sh.top[t] : 0;
    if (cluster > 1) {
        // the first CTA's first warp joins the parts: lane c has list c, which is in order, and
        // the largest head is taken k times
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (rank == 0 && t < 32) {
            for (int r = 1; r < cluster; r++) all = join(all, cl.map_shared_rank(&sh, r)->all);
            const Shared* theirs = cl.map_shared_rank(&sh, min(lane, cluster - 1));
            Key head = lane < cluster && k ? theirs->top[0] : 0;
            int at = 0;
            for (int i = 0; i < k; i++) {
                const Key top = warp_max_key(head);
                if (lane == i) key = top;
                if (head == top && head) head = ++at < k ? theirs->top[at] : 0;
            }
        }
        cl.sync();  // no CTA leaves while its list is read
        if (rank) return;
    }
    const float ls = all.s > 0.0f ? logf(all.s) : NAN;
    auto logprob = [&](float x) { return (x - all.m) - ls; };
    if (t == 0) {
        if (a.targets) {
            const int id = a.targets[m_row];
            a.target_logprob[m_row] = id < 0 || id >= a.V ? NAN : logprob(to_f32(row.p[id]));
        }
        if (a.entropy) a.entropy[m_row] = ls - all.w / all.s;
    }
    if (t < k) {
        a.top_ids[m_row * k + t] = key_number(key);
        a.top_logprob[m_row * k + t] = logprob(key_value(key));
    }
}

template <typename T>
cudaError_t launch_t(const LogprobArgs& a, cudaStream_t s) {
    // More CTAs to a row while it has over 4096 elements for each and the grid stays within two
    // CTAs to an SM: few rows are bound by latency (1 x 32000: 8.4 us with one CTA, 6.8 with 8;
    // 16 x 128256: 15.8, 9.7), more of them by what each CTA has to join (64 x 32000: 9.1 us
    // with 4, 10.4 with 8; 128 x 128256: 21.6, 17.8, 19.5 with 1, 2, 4), many by memory (2048 x
    // 128256: 114 us with 1, 150 with 2).
    int cluster = 1;
    while (cluster < kMaxCluster && a.V / cluster > 4096 && (int64_t)a.M * cluster <= 148) cluster *= 2;
    count_launch();
    return launch_ex(logprob_kernel<T>, dim3((unsigned)((int64_t)a.M * cluster)), dim3(kThreads), 0, s, (unsigned)cluster, a, cluster);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, cudaStream_t s) {
    if (a.dtype == kF32) return launch_t<float>(a, s);
    return a.dtype == kBF16 ? launch_t<__nv_bfloat16>(a, s) : launch_t<__half>(a, s);
}

}  // namespace nitro
