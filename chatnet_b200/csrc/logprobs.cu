// logprobs.cu -- log probabilities of given tokens with the distribution's
// entropy and its most likely alternatives (cn_logprobs_dev), so a host that
// reports or scores tokens need not copy the logits back.
//
//   m = max x, S = sum e^(x - m), T = sum (x - m) e^(x - m)
//   logprob(t) = x_t - m - log S,   entropy = log S - T / S
#include <float.h>

#include "cn_common.cuh"
#include "cn_internal.h"
#include "kvq4.cuh"

namespace cn {

namespace {

constexpr int kMaxTop = 64;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// An order on (value, lower index first) as one whole number: larger values
// first, NaN after everything.
__device__ __forceinline__ uint64_t order_key(float v, int i) {
    const uint32_t u = __float_as_uint(v + 0.f);  // -0 as +0
    const uint32_t o = v != v ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((uint64_t)o << 32) | (0xFFFFFFFFu - (uint32_t)i);
}

__device__ __forceinline__ uint64_t warp_max_u64(uint64_t k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t x = __shfl_xor_sync(0xffffffffu, k, o);
        k = x > k ? x : k;
    }
    return k;
}

}  // namespace

// One CTA per row, three passes, then one pass per alternative.
template <typename T>
__global__ void __launch_bounds__(256)
    logprobs_plain_kernel(const T* __restrict__ logits, int64_t stride, int n, const int* __restrict__ tokens, int top,
                          float* __restrict__ logprob, float* __restrict__ entropy, int* __restrict__ top_ids,
                          float* __restrict__ top_lp) {
    __shared__ float red[3][8];
    __shared__ uint64_t best[8];
    const T* x = logits + (int64_t)blockIdx.x * stride;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = -INFINITY;
    bool nan = false;
    for (int i = threadIdx.x; i < n; i += 256) {
        const float v = to_f(x[i]);
        nan |= v != v;
        m = fmaxf(m, v);
    }
    if (nan) m = INFINITY;  // x - inf: every result of the row is NaN or -inf
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!lane) red[0][w] = m;
    __syncthreads();
    for (int k = 0; k < 8; k++) m = fmaxf(m, red[0][k]);
    float S = 0.f, U = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) {
        const float d = to_f(x[i]) - m, e = expf(d);
        S += e;
        if (!(e == 0.f)) U = fmaf(d, e, U);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        S += __shfl_xor_sync(0xffffffffu, S, o);
        U += __shfl_xor_sync(0xffffffffu, U, o);
    }
    if (!lane) {
        red[1][w] = S;
        red[2][w] = U;
    }
    __syncthreads();
    S = U = 0.f;
    for (int k = 0; k < 8; k++) {
        S += red[1][k];
        U += red[2][k];
    }
    const float ls = logf(S);
    if (threadIdx.x == 0) {
        if (entropy) entropy[blockIdx.x] = ls - U / S;
        if (logprob) {
            const int t = tokens[blockIdx.x];
            logprob[blockIdx.x] = t >= 0 && t < n ? (to_f(x[t]) - m) - ls : NAN;
        }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top; k++) {
        uint64_t bk = 0;
        for (int i = threadIdx.x; i < n; i += 256) {
            const uint64_t key = order_key(to_f(x[i]), i);
            if (key < last && key > bk) bk = key;
        }
        bk = warp_max_u64(bk);
        __syncthreads();
        if (!lane) best[w] = bk;
        __syncthreads();
        for (int j = 0; j < 8; j++) bk = best[j] > bk ? best[j] : bk;
        last = bk;
        if (threadIdx.x == 0) {
            const int i = (int)(0xFFFFFFFFu - (uint32_t)bk);
            top_ids[(int64_t)blockIdx.x * top + k] = i;
            if (top_lp) top_lp[(int64_t)blockIdx.x * top + k] = (to_f(x[i]) - m) - ls;
        }
    }
}

int logprobs_launch(cn_ctx* ctx, int type, const void* logits, int64_t stride, int rows, int vocab, const int* tokens,
                    int top, float* logprob, float* entropy, int* top_ids, float* top_lp, cudaStream_t st) {
    if (type == CN_TYPE_F16)
        logprobs_plain_kernel<__half><<<rows, 256, 0, st>>>(static_cast<const __half*>(logits), stride, vocab, tokens,
                                                            top, logprob, entropy, top_ids, top_lp);
    else
        logprobs_plain_kernel<float><<<rows, 256, 0, st>>>(static_cast<const float*>(logits), stride, vocab, tokens,
                                                           top, logprob, entropy, top_ids, top_lp);
    CN_CUDA(cudaGetLastError());
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
    CN_CHECK(row_stride < (1ll << 40), CN_ERR_INVALID_ARG, "row_stride too large");
    CN_CHECK(top_n >= 0 && top_n <= kMaxTop && top_n <= vocab, CN_ERR_INVALID_ARG,
             "top_n %d outside [0, min(%d, vocabulary %d)]", top_n, kMaxTop, vocab);
    CN_CHECK(!d_logprob == !d_tokens, CN_ERR_INVALID_ARG, "tokens and their log probabilities go together");
    CN_CHECK((top_n > 0) == (d_top_ids != nullptr) && (top_n > 0 || !d_top_logprobs), CN_ERR_INVALID_ARG,
             "top_n and the outputs of the alternatives go together");
    CN_CHECK(d_logprob || d_entropy || d_top_ids, CN_ERR_INVALID_ARG, "no output asked for");
    CN_CHECK((uintptr_t)d_logits % (type == CN_TYPE_F16 ? 2 : 4) == 0, CN_ERR_INVALID_ARG, "misaligned logits");
    DeviceScope ds(ctx->device);
    return logprobs_launch(ctx, type, d_logits, row_stride, rows, vocab, d_tokens, top_n, d_logprob, d_entropy,
                           d_top_ids, d_top_logprobs, (cudaStream_t)stream);
}
