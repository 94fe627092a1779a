// logprobs.cu -- log probabilities of given tokens with the distribution's
// entropy and its most likely alternatives (cn_logprobs_dev), so a host that
// reports or scores tokens need not copy the logits back.
//
//   m = max x, S = sum e^(x - m), T = sum (x - m) e^(x - m)
//   logprob(t) = x_t - m - log S,   entropy = log S - T / S
// One pass over the logits: each thread keeps its own m, S and T, which are
// scaled to a common m at the end.  Bound: the logits' bytes, each read once.
//
// The alternatives come out of the same pass.  Order: larger value, then lower
// id, NaN last, as one 64-bit key.  A CTA keeps a buffer of candidates and a
// bound t below which nothing can be among its top n.  t starts from the first
// chunk (each of the W warps finds the k-th largest of its lanes' maxima, k =
// ceil(n / W); the smallest of the W has at least n values at or above it)
// and is the n-th best value whenever the buffer is cut back to n; after the first
// chunks next to nothing passes it.
//
// A row is split over a cluster of CTAs when there are few rows; their sums and
// lists meet in the first CTA's shared memory.  No workspace, no atomics on
// global memory, one launch.
//
// 4096 rows of 32000 fp32: 88 us, 5.9 TB/s (0.92 of a copy's rate).  300 rows of
// 131071 fp16 with 8 alternatives: 40 us, 2.0 TB/s, bound by latency: one CTA a row is two
// CTAs on most SMs and three on four, sixteen warps whose loads, conversions and
// exponentials follow one another (43 % of the issue slots, 24 % of DRAM's rate).  Few rows
// are bound by the choice among the candidates, about 5 us: one row of 32000 with 5 takes
// 9 us, 32 with 20 11.
#include <float.h>

#include "cn_common.cuh"
#include "cn_internal.h"
#include "kvq4.cuh"

namespace cn {

namespace {

constexpr int kMaxTop = 64;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPer = 16;              // values a thread takes at a time
constexpr int kChunk = kThreads * kPer;
constexpr int kCut = 128;             // candidates at which the careful way cuts the buffer back
constexpr int kSmall = 256;           // keys that are ranked by counting
static_assert(kCut >= kMaxTop, "a cut leaves kMaxTop");
constexpr int kBuf = kCut + kChunk;   // (a chunk can add all its values)
constexpr int kMaxCluster = 16;

using Key = unsigned long long;

struct LpArgs {
    const void* logits;
    int64_t stride;
    int n, top;
    const int* tokens;
    float *logprob, *entropy;
    int* top_ids;
    float* top_lp;
};

// A value's place in the order as a whole number (NaN 0).
__device__ __forceinline__ uint32_t order32(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);  // -0 as +0
    return v != v ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
    return o == 0u ? NAN : __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
constexpr uint32_t kMinusInf = 0x007FFFFFu, kZero = 0x80000000u;  // order32 of -inf and 0

// 16 bytes of logits as floats
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int N = 4;
    __device__ static void get(const uint4& u, float* x) {
        x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z),
        x[3] = __uint_as_float(u.w);
    }
    __device__ static uint32_t minus_inf() { return 0xFF800000u; }
};
template <>
struct Vec<__half> {
    static constexpr int N = 8;
    __device__ static void get(const uint4& u, float* x) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    __device__ static uint32_t minus_inf() { return 0xFC00FC00u; }
};

// The running sums of one thread, relative to m; `top` is its largest value.
struct Sums {
    float m = -INFINITY, top = -INFINITY;
    float2 S = {0.f, 0.f}, T = {0.f, 0.f};
    __device__ void raise(float to) {  // to > m
        if (m != -INFINITY) {
            const float d = fmaxf(m - to, -200.f), f = expf(d);  // (0 from there on, and d stays finite)
            T.x = f * fmaf(d, S.x, T.x), T.y = f * fmaf(d, S.y, T.y);
            S.x *= f, S.y *= f;
        }
        m = to;
    }
    // m follows when outgrown by e^4: seldom, and T, which a later m takes d S from,
    // stays within a few S (entropies of 4096 rows of 32000: off by at most 1.2e-6 of
    // them, as with 2 or 8; 4.6e-5 with 16; the time is the same)
    __device__ void see(float v) {
        top = fmaxf(top, v);
        if (v > m + 4.f) raise(v);
    }
    template <int N>
    __device__ void add(const float* x) {
        const float mu = m == -INFINITY ? 0.f : m;
        const float2 nm = make_float2(-mu, -mu);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            float2 d = add2(make_float2(x[i], x[i + 1]), nm);
            // (below e^-200 nothing is left; keeps -inf * 0 out and NaN in)
            d.x = max_nan(d.x, -200.f), d.y = max_nan(d.y, -200.f);
            const float2 l = mul2(d, make_float2(1.44269504088896341f, 1.44269504088896341f));
            const float2 e = make_float2(ex2(l.x), ex2(l.y));
            S = add2(S, e);
            T = fma2(d, e, T);
        }
    }
};

// Brings sums over [m, S, T] to their common maximum; every lane gets them.
__device__ __forceinline__ void join(float& m, float& S, float& T, float m2, float S2, float T2) {
    const float M = fmaxf(m, m2);
    auto scale = [&](float& s, float& t, float mi) {
        if (mi != M && mi != -INFINITY) {
            const float d = fmaxf(mi - M, -200.f), f = expf(d);
            t = f * fmaf(d, s, t);
            s *= f;
        }
    };
    scale(S, T, m);
    scale(S2, T2, m2);
    m = M;
    S += S2;
    T += T2;
}

__device__ __forceinline__ Key warp_max(Key k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Key x = __shfl_xor_sync(0xffffffffu, k, o);
        k = x > k ? x : k;
    }
    return k;
}

// Shared memory of best_keys.
struct Pick {
    Key list[kMaxTop];   // the result
    Key few[kSmall];
    Key red[2 * kWarps];
    uint32_t bound[kWarps];
    int count;
};

// The `top` largest of buf[0..cnt), largest first, into s.list (0 where there
// are fewer).  Whole CTA; buf must be visible (a barrier before).  Many keys are
// first brought down by a bound as in the first chunk, few are ranked by
// counting the larger ones, and many equal values (the bound lets them all
// through) go one after another.
__device__ void best_keys(const Key* buf, int cnt, int top, Pick& s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < top) s.list[tid] = 0;
    if (tid == 0) s.count = 0;
    const Key* from = buf;
    bool rank = cnt <= kSmall;
    if (!rank) {
        uint32_t w = 0, last = 0;
        for (int i = tid; i < cnt; i += kThreads) w = max(w, (uint32_t)(buf[i] >> 32));
        for (int r = 0; r < (top + kWarps - 1) / kWarps; r++) {  // (cnt > kThreads: every lane has a key)
            last = __reduce_max_sync(0xffffffffu, w);
            if (lane == __ffs(__ballot_sync(0xffffffffu, w == last)) - 1) w = 0;
        }
        if (lane == 0) s.bound[warp] = last;
        __syncthreads();
        uint32_t t = s.bound[0];
#pragma unroll
        for (int i = 1; i < kWarps; i++) t = min(t, s.bound[i]);
        for (int i = tid; i < cnt; i += kThreads) {
            const Key k = buf[i];
            if ((uint32_t)(k >> 32) >= t) {
                const int at = atomicAdd(&s.count, 1);
                if (at < kSmall) s.few[at] = k;
            }
        }
        __syncthreads();
        if (s.count <= kSmall) {
            rank = true;
            from = s.few;
            cnt = s.count;
        }
    } else {
        __syncthreads();
    }
    if (rank) {
        if (tid < cnt) {
            const Key k = from[tid];
            int r = 0;
#pragma unroll 4
            for (int j = 0; j < cnt; j++) r += from[j] > k;
            if (r < top) s.list[r] = k;
        }
    } else {
        // a thread looks again only when its own was taken
        auto mine = [&](Key below) {
            Key b = 0;
            for (int i = tid; i < cnt; i += kThreads) {
                const Key k = buf[i];
                if (k < below && k > b) b = k;
            }
            return b;
        };
        Key own = mine(~0ull);
        for (int r = 0; r < top; r++) {
            const Key w = warp_max(own);
            if (lane == 0) s.red[(r & 1) * kWarps + warp] = w;
            __syncthreads();
            Key k = 0;
#pragma unroll
            for (int i = 0; i < kWarps; i++) {
                const Key x = s.red[(r & 1) * kWarps + i];
                k = x > k ? x : k;
            }
            if (tid == 0) s.list[r] = k;
            if (k != 0 && own == k) own = mine(k);
        }
    }
    __syncthreads();
}

}  // namespace

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const LpArgs a) {
    constexpr int VN = Vec<T>::N, U = kPer / VN;
    extern __shared__ __align__(16) uint8_t smem[];         // (TOP)
    Key* buf = reinterpret_cast<Key*>(smem);                // [kBuf]
    Key* meet = buf + kBuf;                                 // [kMaxCluster][kMaxTop] the CTAs' lists (first CTA)
    Pick& pick = *reinterpret_cast<Pick*>(meet + kMaxCluster * kMaxTop);
    uint32_t* bound = pick.bound;
    Key* list = pick.list;
    __shared__ float red[kWarps][3];
    __shared__ float sums[kMaxCluster][3];
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t cs = cluster_size(), rank = cluster_rank();
    const int64_t row = blockIdx.x / cs;
    if (cs > 1) cluster_arrive_relaxed();
    if (TOP && tid == 0) s_count = 0;
    const T* x0 = static_cast<const T*>(a.logits) + row * a.stride;
    float xt = NAN;
    if (rank == 0 && tid == 0 && a.logprob) {
        const int t = a.tokens[row];
        if (t >= 0 && t < a.n) xt = (float)x0[t];
    }
    // the row in 16-byte pieces from the boundary at or before its start; this
    // CTA's share of them
    const int off = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    const uint4* v = reinterpret_cast<const uint4*>(x0 - off);
    const int pieces = (int)(((int64_t)off + a.n + VN - 1) / VN);
    const int v0 = (int)((int64_t)pieces * rank / cs), v1 = (int)((int64_t)pieces * (rank + 1) / cs);
    // pieces within the row as a whole
    const int in0 = max(v0, off ? 1 : 0), in1 = min(v1, (int)(((int64_t)off + a.n) / VN));
    auto load_chunk = [&](uint4(&to)[U], int q) {
        const int b = v0 + q * U * kThreads;
        if (b >= in0 && b + U * kThreads <= in1) {
            const uint4* p = v + b + tid;
#pragma unroll
            for (int k = 0; k < U; k++) to[k] = __ldcs(p + k * kThreads);
            return;
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int i = b + k * kThreads + tid;
            to[k] = make_uint4(Vec<T>::minus_inf(), Vec<T>::minus_inf(), Vec<T>::minus_inf(), Vec<T>::minus_inf());
            if (i >= in0 && i < in1) {
                to[k] = __ldcs(v + i);
            } else if (i < v1) {  // the row's first or last piece
                T* p = reinterpret_cast<T*>(&to[k]);
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    const int e = i * VN - off + j;
                    if (e >= 0 && e < a.n) p[j] = x0[e];
                }
            }
        }
    };
    Sums sm;
    // Candidates are the values above the float t (in the order: above t_ord).
    // They go into buf as they come; the buffer is cut back to the best after
    // chunks 0, 4, 16, 64 and so on, which leaves it far from full unless the
    // row rises along its length.  Then, or where no t tells NaN or -inf apart, the
    // CTA's share is gone through again chunk by chunk.
    uint32_t t_ord = 0;
    float t = INFINITY;
    bool again = false;
    auto take = [&](const uint4(&cur)[U]) {
        float cm = -INFINITY;
#pragma unroll
        for (int k = 0; k < U; k++) {
            float x[VN];
            Vec<T>::get(cur[k], x);
#pragma unroll
            for (int i = 0; i < VN; i++) cm = fmaxf(cm, x[i]);
        }
        sm.see(cm);
#pragma unroll
        for (int k = 0; k < U; k++) {
            float x[VN];
            Vec<T>::get(cur[k], x);
            sm.template add<VN>(x);
        }
        return cm;
    };
    auto keep = [&](const uint4(&cur)[U], int c) {
#pragma unroll
        for (int k = 0; k < U; k++) {
            float x[VN];
            Vec<T>::get(cur[k], x);
            const int e = (v0 + (c * U + k) * kThreads + tid) * VN - off;
#pragma unroll
            for (int i = 0; i < VN; i++)
                if (x[i] > t) {
                    const int at = atomicAdd(&s_count, 1);
                    if (at < kBuf) buf[at] = ((Key)order32(x[i]) << 32) | (0xFFFFFFFFu - (uint32_t)(e + i));
                }
        }
    };
    // (whole CTA, after a barrier)
    auto cut = [&]() {
        const int cnt = s_count;
        if (cnt > a.top && cnt <= kBuf) {
            best_keys(buf, cnt, a.top, pick);
            if (tid < a.top) buf[tid] = list[tid];
            if (tid == 0) s_count = a.top;
            // (what comes later has higher ids: an equal value is not better)
            t_ord = (uint32_t)(list[a.top - 1] >> 32);
            t = order_value(t_ord);
        }
        __syncthreads();
    };
    const int chunks = (v1 - v0 + U * kThreads - 1) / (U * kThreads);
    // (a CTA keeps 16 KB of loads in flight: one chunk of fp32, two of fp16)
    constexpr int AHEAD = VN / 4;
    uint4 ring[AHEAD + 1][U];
#pragma unroll
    for (int q = 0; q <= AHEAD; q++) load_chunk(ring[q], q);
    {
        const float cm = take(ring[0]);
        if constexpr (TOP) {
            // (of the warps whose lanes all have values)
            const int warps = min(v1 - v0, kThreads) / 32;
            const int rounds = warps ? (a.top + warps - 1) / warps : 33;
            if (rounds <= 32) {
                uint32_t w = order32(cm), last = 0;
                for (int r = 0; r < rounds; r++) {
                    last = __reduce_max_sync(0xffffffffu, w);
                    if (lane == __ffs(__ballot_sync(0xffffffffu, w == last)) - 1) w = 0;
                }
                if (lane == 0) bound[warp] = warp < warps ? last : 0xFFFFFFFFu;
            }
            __syncthreads();
            if (rounds <= 32) {
                t_ord = bound[0];
#pragma unroll
                for (int i = 1; i < kWarps; i++) t_ord = min(t_ord, bound[i]);
            }
            again = t_ord <= kMinusInf;  // (a maximum of -inf may stand for NaN or nothing)
            if (!again) {
                t_ord -= t_ord == kZero ? 2 : 1;  // the next value below (0 and -0 are one)
                t = order_value(t_ord);
                if (cm > t) keep(ring[0], 0);
                if (chunks > 1) {
                    __syncthreads();
                    cut();
                }
            }
        }
    }
    for (int c = 1; c < chunks; c++) {
#pragma unroll
        for (int q = 0; q < AHEAD; q++)
#pragma unroll
            for (int k = 0; k < U; k++) ring[q][k] = ring[q + 1][k];
        if (c + AHEAD < chunks) load_chunk(ring[AHEAD], c + AHEAD);
        const float cm = take(ring[0]);
        if constexpr (TOP) {
            if (cm > t) keep(ring[0], c);
            if ((c & (c - 1)) == 0 && (c & 0x55555554)) {  // 4, 16, 64, ...
                __syncthreads();
                cut();
            }
        }
    }
    if constexpr (TOP) {
        __syncthreads();
        if (again || s_count > kBuf) {
            __syncthreads();
            if (tid == 0) s_count = 0;
            bool full = false;  // (as many as asked for are kept: only larger values count)
            __syncthreads();
            for (int c = 0; c < chunks; c++) {
                for (int h = 0; h < kPer; h++) {
                    const int i = v0 + (c * U + h / VN) * kThreads + tid, e = i * VN - off + h % VN;
                    if (e < 0 || e >= a.n || i >= v1) continue;
                    const uint32_t o = order32((float)x0[e]);
                    if (!full || o > t_ord) buf[atomicAdd(&s_count, 1)] = ((Key)o << 32) | (0xFFFFFFFFu - (uint32_t)e);
                }
                if (__syncthreads_or(*(volatile int*)&s_count > kCut)) {
                    full = true;  // (kCut is above any top)
                    cut();
                }
            }
            __syncthreads();
        }
    }
    if (sm.top > sm.m) sm.raise(sm.top);
    // the CTA's sums
    float m = sm.m, S = sm.S.x + sm.S.y, Tt = sm.T.x + sm.T.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        join(m, S, Tt, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, S, o),
             __shfl_xor_sync(0xffffffffu, Tt, o));
    if (lane == 0) {
        red[warp][0] = m;
        red[warp][1] = S;
        red[warp][2] = Tt;
    }
    __syncthreads();
    if (TOP) best_keys(buf, s_count, a.top, pick);
    if (warp == 0) {
        const int w = lane < kWarps ? lane : 0;
        m = lane < kWarps ? red[w][0] : -INFINITY;
        S = lane < kWarps ? red[w][1] : 0.f;
        Tt = lane < kWarps ? red[w][2] : 0.f;
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1)
            join(m, S, Tt, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, S, o),
                 __shfl_xor_sync(0xffffffffu, Tt, o));
    }
    if (cs > 1) {
        // to the first CTA
        __syncwarp();
        cluster_wait();  // (it has started)
        if (tid == 0) {
            const uint32_t d = map_rank(smem_u32(&sums[rank][0]), 0);
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(d), "f"(m) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(d + 4), "f"(S) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(d + 8), "f"(Tt) : "memory");
        }
        if (TOP && tid < a.top)
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_rank(smem_u32(&meet[rank * a.top + tid]), 0)),
                         "l"(list[tid])
                         : "memory");
        __syncwarp();
        cluster_arrive();
        if (rank != 0) return;
        cluster_wait();
        if (warp == 0) {
            m = lane < (int)cs ? sums[lane & (kMaxCluster - 1)][0] : -INFINITY;
            S = lane < (int)cs ? sums[lane & (kMaxCluster - 1)][1] : 0.f;
            Tt = lane < (int)cs ? sums[lane & (kMaxCluster - 1)][2] : 0.f;
#pragma unroll
            for (int o = kMaxCluster / 2; o > 0; o >>= 1)
                join(m, S, Tt, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, S, o),
                     __shfl_xor_sync(0xffffffffu, Tt, o));
        }
        if (TOP) best_keys(meet, (int)cs * a.top, a.top, pick);
    }
    if (tid == 0) {
        const float ls = m == -INFINITY ? NAN : logf(S);
        if (a.entropy) a.entropy[row] = ls - Tt / S;
        if (a.logprob) a.logprob[row] = (xt - m) - ls;
        red[0][0] = m;
        red[0][1] = ls;
    }
    if (TOP) {
        __syncthreads();
        if (tid < a.top) {
            const Key k = list[tid];
            a.top_ids[row * a.top + tid] = (int)(0xFFFFFFFFu - (uint32_t)k);
            if (a.top_lp) a.top_lp[row * a.top + tid] = (order_value((uint32_t)(k >> 32)) - red[0][0]) - red[0][1];
        }
    }
}

int logprobs_launch(cn_ctx* ctx, int type, const void* logits, int64_t stride, int rows, int vocab, const int* tokens,
                    int top, float* logprob, float* entropy, int* top_ids, float* top_lp, cudaStream_t st) {
    LpArgs a{logits, stride, vocab, top, tokens, logprob, entropy, top_ids, top_lp};
    using Fn = void (*)(LpArgs);
    const bool half = type == CN_TYPE_F16;
    const Fn fn = half ? (top ? (Fn)logprobs_kernel<__half, true> : (Fn)logprobs_kernel<__half, false>)
                       : (top ? (Fn)logprobs_kernel<float, true> : (Fn)logprobs_kernel<float, false>);
    const size_t smem = top ? (kBuf + kMaxCluster * kMaxTop) * sizeof(Key) + sizeof(Pick) : 0;
    // CTAs per row: as many as give every SM two (32 rows of 32000 with 20
    // alternatives: 13.2 us with 2, 9.8 with 8, 14 with 16), and at least a quarter
    // of a chunk for each
    const int64_t room = (int64_t)ctx->sms * 2;
    int cluster = 1;
    while (cluster < kMaxCluster && 2 * (int64_t)cluster * rows <= room && 2 * cluster * (kChunk / 4) <= vocab)
        cluster *= 2;
    CN_CHECK((int64_t)rows * cluster < (1ll << 31), CN_ERR_INVALID_ARG, "too many rows (%d)", rows);
    const uint32_t bit = 1u << (16 + (half ? 2 : 0) + (top ? 1 : 0));
    if (!(__atomic_load_n(&ctx->kvq4_ready, __ATOMIC_RELAXED) & bit)) {
        CN_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        CN_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        __atomic_fetch_or(&ctx->kvq4_ready, bit, __ATOMIC_RELAXED);
    }
    CN_CUDA(launch_cluster_k(false, cluster, fn, dim3((unsigned)(rows * cluster)), dim3(kThreads), smem, st, a));
    return CN_OK;
}

int logprobs_check(int vocab, const void* tokens, int top, const void* logprob, const void* entropy,
                   const void* top_ids, const void* top_lp) {
    CN_CHECK(top >= 0 && top <= kMaxTop && top <= vocab, CN_ERR_INVALID_ARG,
             "top_n %d outside [0, min(%d, vocabulary %d)]", top, kMaxTop, vocab);
    CN_CHECK(!logprob == !tokens, CN_ERR_INVALID_ARG, "tokens and their log probabilities go together");
    CN_CHECK((top > 0) == (top_ids != nullptr) && (top > 0 || !top_lp), CN_ERR_INVALID_ARG,
             "top_n and the outputs of the alternatives go together");
    CN_CHECK(logprob || entropy || top_ids, CN_ERR_INVALID_ARG, "no output asked for");
    return CN_OK;
}

}  // namespace cn

using namespace cn;

extern "C" int cn_logprobs_dev(cn_ctx* ctx, int type, const void* d_logits, int64_t row_stride, int rows, int vocab,
                               const int* d_tokens, int top_n, float* d_logprob, float* d_entropy, int* d_top_ids,
                               float* d_top_logprobs, void* stream) {
    CN_CHECK(ctx && d_logits, CN_ERR_INVALID_ARG, "null argument");
    CN_CHECK(type == CN_TYPE_F32 || type == CN_TYPE_F16, CN_ERR_UNSUPPORTED, "logits of type %d (F32 or F16)", type);
    CN_CHECK(rows >= 1 && vocab >= 1 && row_stride >= vocab, CN_ERR_INVALID_ARG,
             "bad shape (%d rows, vocabulary %d, stride %lld)", rows, vocab, (long long)row_stride);
    CN_CHECK(row_stride < (1ll << 40) && vocab < (1 << 30), CN_ERR_INVALID_ARG, "row too large");
    int rc = logprobs_check(vocab, d_tokens, top_n, d_logprob, d_entropy, d_top_ids, d_top_logprobs);
    if (rc) return rc;
    CN_CHECK((uintptr_t)d_logits % (type == CN_TYPE_F16 ? 2 : 4) == 0, CN_ERR_INVALID_ARG, "misaligned logits");
    DeviceScope ds(ctx->device);
    return logprobs_launch(ctx, type, d_logits, row_stride, rows, vocab, d_tokens, top_n, d_logprob, d_entropy,
                           d_top_ids, d_top_logprobs, (cudaStream_t)stream);
}
