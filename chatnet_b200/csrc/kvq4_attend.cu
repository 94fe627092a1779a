// kvq4_attend.cu -- attention over the 4-bit KV cache (cn_kvq4_attend_dev).
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale (q . k_p) - max)
// over positions p = 0 .. pos[b] + i of token i, with one pass over the cache
// (running maximum and sum, fp32).
#include "kvq4.cuh"

namespace cn {

// One warp per (token, query head): lane (g = lane >> 2, t = lane & 3) holds
// values 32 b + 8 t + g of every block, i.e. nibble t of the pieces of chunk g.
template <int NB>
__global__ void __launch_bounds__(128)
    kvq4_attend_plain_kernel(const float* __restrict__ q, int64_t q_stride, float* __restrict__ out, int64_t out_stride,
                             const int* __restrict__ pos, const int* __restrict__ count, int n_new, int n_heads,
                             int n_kv, int64_t n_rows, float scale, const float2* __restrict__ rope, int neox,
                             const uint8_t* __restrict__ kq, const __half* __restrict__ kd,
                             const uint8_t* __restrict__ vq, const __half* __restrict__ vd, int64_t seq_rows,
                             int ctx_len) {
    constexpr int HD = 32 * NB;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= n_rows) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int h = (int)(row % n_heads);
    const int64_t tok = row / n_heads;
    const int b = (int)(tok / n_new), i = (int)(tok % n_new);
    int p0;
    if (i >= kvq4_active(pos, count, b, n_new, ctx_len, p0)) return;
    const int len = p0 + i + 1;
    float x[NB], o[NB];
    const float* qr = q + tok * q_stride + (int64_t)h * HD;
    const float2* tab = rope + (int64_t)(p0 + i) * (HD / 2);
#pragma unroll
    for (int j = 0; j < NB; j++) {
        const int e = 32 * j + 8 * t + g;
        o[j] = 0.f;
        if (!rope) {
            x[j] = qr[e];
        } else if (neox) {
            const float2 cs = tab[e % (HD / 2)];
            x[j] = e < HD / 2 ? __fsub_rn(__fmul_rn(qr[e], cs.x), __fmul_rn(qr[e + HD / 2], cs.y))
                              : __fadd_rn(__fmul_rn(qr[e - HD / 2], cs.y), __fmul_rn(qr[e], cs.x));
        } else {
            const float2 cs = tab[e / 2];
            x[j] = (e & 1) ? __fadd_rn(__fmul_rn(qr[e - 1], cs.y), __fmul_rn(qr[e], cs.x))
                           : __fsub_rn(__fmul_rn(qr[e], cs.x), __fmul_rn(qr[e + 1], cs.y));
        }
    }
    const int64_t base = (int64_t)b * seq_rows + (int64_t)(h / (n_heads / n_kv)) * ctx_len;
    float m = -INFINITY, l = 0.f;
    for (int p = 0; p < len; p++) {
        const int64_t r = base + p;
        const uint16_t* kr = reinterpret_cast<const uint16_t*>(kq + r * (HD / 2) + g * (2 * NB));
        const uint16_t* vr = reinterpret_cast<const uint16_t*>(vq + r * (HD / 2) + g * (2 * NB));
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NB; j++)
            s = fmaf(x[j], __half2float(kd[r * NB + j]) * (float)((int)((kr[j] >> (4 * t)) & 15) - 8), s);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
        s *= scale;
        const float mn = fmaxf(m, s), a = expf(m - mn), w = expf(s - mn);
        l = fmaf(l, a, w);
#pragma unroll
        for (int j = 0; j < NB; j++)
            o[j] = fmaf(o[j], a, w * (__half2float(vd[r * NB + j]) * (float)((int)((vr[j] >> (4 * t)) & 15) - 8)));
        m = mn;
    }
    float* dst = out + tok * out_stride + (int64_t)h * HD;
#pragma unroll
    for (int j = 0; j < NB; j++) dst[32 * j + 8 * t + g] = o[j] / l;
}

int kvq4_attend(cn_ctx* ctx, const cn_kvq4& c, const float* q, int64_t q_stride, float* out, int64_t out_stride,
                const int* pos, const int* count, int batch, int n_new, int n_heads, float scale, const float2* rope,
                int neox, cudaStream_t st) {
    const int64_t rows = (int64_t)batch * n_new * n_heads, ctas = (rows + 3) / 4;
    CN_CHECK(ctas < (1ll << 31), CN_ERR_INVALID_ARG, "too many rows (%lld)", (long long)rows);
#define CALL(NB)                                                                                                   \
    kvq4_attend_plain_kernel<NB><<<(unsigned)ctas, 128, 0, st>>>(                                                  \
        q, q_stride, out, out_stride, pos, count, n_new, n_heads, c.n_kv_heads, rows, scale, rope, neox,           \
        static_cast<const uint8_t*>(c.k_quants), static_cast<const __half*>(c.k_scales),                           \
        static_cast<const uint8_t*>(c.v_quants), static_cast<const __half*>(c.v_scales), kvq4_seq_rows(c),         \
        c.ctx_len);                                                                                                \
    break
    switch (c.head_dim) {
        case 32: CALL(1);
        case 64: CALL(2);
        case 96: CALL(3);
        case 128: CALL(4);
        default: CALL(8);
    }
#undef CALL
    CN_CUDA(cudaGetLastError());
    return CN_OK;
}

}  // namespace cn

using namespace cn;

extern "C" int cn_kvq4_attend_dev(cn_ctx* ctx, const cn_kvq4* cache, const float* d_q, int64_t q_stride, float* d_out,
                                  int64_t out_stride, const int* d_pos, const int* d_count, int batch, int n_new,
                                  int n_heads, float scale, const float* d_rope, int rope_neox, void* stream) {
    int rc = kvq4_check(ctx, cache, batch, n_new);
    if (rc) return rc;
    CN_CHECK(d_q && d_out && d_pos, CN_ERR_INVALID_ARG, "null argument");
    CN_CHECK(n_heads >= 1 && n_heads % cache->n_kv_heads == 0, CN_ERR_INVALID_ARG,
             "n_heads %d is not a multiple of n_kv_heads %d", n_heads, cache->n_kv_heads);
    const int64_t qd = (int64_t)n_heads * cache->head_dim;
    CN_CHECK(q_stride >= qd && out_stride >= qd && q_stride % 4 == 0 && out_stride % 4 == 0, CN_ERR_INVALID_ARG,
             "q_stride %lld / out_stride %lld: at least %lld values and a multiple of 4", (long long)q_stride,
             (long long)out_stride, (long long)qd);
    CN_CHECK(((uintptr_t)d_q | (uintptr_t)d_out) % 16 == 0 && (uintptr_t)d_rope % 8 == 0, CN_ERR_INVALID_ARG,
             "q and out must be 16-byte aligned, the rope table 8-byte");
    CN_CHECK(isfinite(scale) && scale > 0.f, CN_ERR_INVALID_ARG, "scale must be finite and positive");
    CN_CHECK(rope_neox == 0 || rope_neox == 1, CN_ERR_INVALID_ARG, "rope_neox is 0 or 1");
    DeviceScope ds(ctx->device);
    return kvq4_attend(ctx, *cache, d_q, q_stride, d_out, out_stride, d_pos, d_count, batch, n_new, n_heads, scale,
                       reinterpret_cast<const float2*>(d_rope), rope_neox, (cudaStream_t)stream);
}
