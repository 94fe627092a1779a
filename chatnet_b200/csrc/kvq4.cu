// kvq4.cu -- writing new rows into the 4-bit KV cache and reading rows back
// (cn_kvq4_append_dev, cn_kvq4_read_dev).
//
// Append, per row and block of 32 values (all in fp32, each step rounded):
//   x limited to +-8 * 65504, NaN taken as 0;
//   m = min(x) if -min(x) >= max(x) else max(x);  d = fp16(-m / 8)
//   q = the level whose value d * (q - 8) is nearest to x, halves up, in
//       0..15 (all 8 where d is 0).
// k rows are rotated first when a RoPE table is given, with the arithmetic of
// the decode attention (ApplyRoPE, TensorMath.cs:418-470; split-half pairs:
// TensorMath.cs:475).
#include "kvq4.cuh"

namespace cn {

namespace {

constexpr int kRowThreads = 256;  // 8 lanes a row: 32 rows per CTA
constexpr float kMaxX = 524032.f;  // 8 * 65504

__device__ __forceinline__ float tame(float x) {
    return x == x ? fminf(fmaxf(x, -kMaxX), kMaxX) : 0.f;
}

// The nearest level to x / d, halves up.  floor(x / d + 8.5) is off by one at
// most (the reciprocal, product and sum are each rounded), so the borders
// d * (q - 8.5) and d * (q - 7.5), exact in fp32 (11 + 5 bits), decide.
__device__ __forceinline__ uint32_t level(float x, float d, float inv) {
    float q = floorf(__fadd_rn(__fmul_rn(x, inv), 8.5f));
    q = fminf(fmaxf(q, 0.f), 15.f);
    const float s = d < 0.f ? -x : x, a = fabsf(d);
    if (q < 15.f && s >= __fmul_rn(a, q - 7.5f)) q += 1.f;
    else if (q > 0.f && s < __fmul_rn(a, q - 8.5f)) q -= 1.f;
    return (uint32_t)(int)q;
}

}  // namespace

// Eight lanes a row: lane g holds the values 32 b + 8 i + g, so a block's
// minimum and maximum need three shuffles for four rows at once, a lane's
// values are exactly the nibbles of its chunk, and a load instruction still
// fetches whole 32-byte sectors.
template <int NB>
__global__ void __launch_bounds__(kRowThreads)
    kvq4_append_kernel(const float* __restrict__ k, const float* __restrict__ v, int64_t kv_stride,
                       const int* __restrict__ pos, const int* __restrict__ count, int n_new, int n_kv,
                       int64_t n_rows, const float2* __restrict__ rope, int neox, uint8_t* __restrict__ kq,
                       __half* __restrict__ kd, uint8_t* __restrict__ vq, __half* __restrict__ vd, int64_t seq_rows,
                       int ctx_len) {
    constexpr int HD = 32 * NB;
    const int g = threadIdx.x & 7;
    const int64_t r = (int64_t)blockIdx.x * (kRowThreads / 8) + (threadIdx.x >> 3);
    const bool is_v = blockIdx.y != 0;
    bool live = r < n_rows && (is_v ? v : k) != nullptr;
    int64_t tok = 0, dst = 0;
    int h = 0, p = 0;
    if (live) {
        h = (int)(r % n_kv);
        tok = r / n_kv;
        const int b = (int)(tok / n_new), i = (int)(tok % n_new);
        int p0;
        live = i < kvq4_active(pos, count, b, n_new, ctx_len, p0);
        p = p0 + i;
        dst = (int64_t)b * seq_rows + (int64_t)h * ctx_len + p;
    }
    float x[NB][4];
    if (live) {
        const float* src = (is_v ? v : k) + tok * kv_stride + (int64_t)h * HD + g;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[b][i] = src[32 * b + 8 * i];
    } else {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[b][i] = 0.f;
    }
    if (!is_v && rope) {
        const float2* tab = rope + (int64_t)p * (HD / 2);  // (p = 0 for a row that is not live)
        if (neox) {
            // e pairs with e + hd/2: a lane holds both (hd/2 is a multiple of 16)
#pragma unroll
            for (int n = 0; n < 2 * NB; n++) {
                const int e0 = n, e1 = n + 2 * NB;  // in units of 8 values
                const float2 cs = tab[8 * n + g];
                float &a = x[e0 / 4][e0 % 4], &c = x[e1 / 4][e1 % 4];
                const float ra = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(c, cs.y));
                const float rc = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(c, cs.x));
                a = ra;
                c = rc;
            }
        } else {
#pragma unroll
            for (int n = 0; n < 4 * NB; n++) {
                const float own = x[n / 4][n % 4];
                const float oth = __shfl_xor_sync(0xffffffffu, own, 1);
                const float2 cs = tab[4 * n + (g >> 1)];
                x[n / 4][n % 4] = (g & 1) ? __fadd_rn(__fmul_rn(oth, cs.y), __fmul_rn(own, cs.x))
                                          : __fsub_rn(__fmul_rn(own, cs.x), __fmul_rn(oth, cs.y));
            }
        }
    }
    uint32_t piece[NB];
    float scale[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[b][i] = tame(x[b][i]);
            lo = i ? fminf(lo, x[b][i]) : x[b][i];
            hi = i ? fmaxf(hi, x[b][i]) : x[b][i];
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const float d = __half2float(__float2half_rn(__fmul_rn(-lo >= hi ? lo : hi, -0.125f)));
        const float inv = d == 0.f ? 0.f : __frcp_rn(d);  // (inv 0: level 8 for every value)
        scale[b] = d;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) w |= (d == 0.f ? 8u : level(x[b][i], d, inv)) << (4 * i);
        piece[b] = w;
    }
    if (!live) return;
    uint8_t* q = (is_v ? vq : kq) + dst * (HD / 2) + g * (2 * NB);
    if constexpr (NB == 8) {
        *reinterpret_cast<uint4*>(q) = make_uint4(piece[0] | piece[1] << 16, piece[2] | piece[3] << 16,
                                                  piece[4] | piece[5] << 16, piece[6] | piece[7] << 16);
    } else if constexpr (NB == 4) {
        *reinterpret_cast<uint2*>(q) = make_uint2(piece[0] | piece[1] << 16, piece[2] | piece[3] << 16);
    } else if constexpr (NB == 2) {
        *reinterpret_cast<uint32_t*>(q) = piece[0] | piece[1] << 16;
    } else {
#pragma unroll
        for (int b = 0; b < NB; b++) reinterpret_cast<uint16_t*>(q)[b] = (uint16_t)piece[b];
    }
    __half* d = (is_v ? vd : kd) + dst * NB;
#pragma unroll
    for (int b = 0; b < NB; b++)
        if (g == b) d[b] = __float2half_rn(scale[b]);
}

template <int NB>
__global__ void __launch_bounds__(kRowThreads)
    kvq4_read_kernel(float* __restrict__ k, float* __restrict__ v, int64_t kv_stride, const int* __restrict__ pos,
                     const int* __restrict__ count, int n_new, int n_kv, int64_t n_rows, const uint8_t* __restrict__ kq,
                     const __half* __restrict__ kd, const uint8_t* __restrict__ vq, const __half* __restrict__ vd,
                     int64_t seq_rows, int ctx_len) {
    constexpr int HD = 32 * NB;
    const int g = threadIdx.x & 7;
    const int64_t r = (int64_t)blockIdx.x * (kRowThreads / 8) + (threadIdx.x >> 3);
    const bool is_v = blockIdx.y != 0;
    float* out = is_v ? v : k;
    if (r >= n_rows || !out) return;
    const int h = (int)(r % n_kv);
    const int64_t tok = r / n_kv;
    const int b = (int)(tok / n_new), i = (int)(tok % n_new);
    int p0;
    if (i >= kvq4_active(pos, count, b, n_new, ctx_len, p0)) return;
    const int64_t src = (int64_t)b * seq_rows + (int64_t)h * ctx_len + p0 + i;
    const uint16_t* q = reinterpret_cast<const uint16_t*>((is_v ? vq : kq) + src * (HD / 2) + g * (2 * NB));
    const __half* d = (is_v ? vd : kd) + src * NB;
    out += tok * kv_stride + (int64_t)h * HD + g;
#pragma unroll
    for (int bl = 0; bl < NB; bl++) {
        const uint32_t w = q[bl];
        const float s = __half2float(d[bl]);
#pragma unroll
        for (int j = 0; j < 4; j++) out[32 * bl + 8 * j] = s * (float)((int)((w >> (4 * j)) & 15u) - 8);
    }
}

int kvq4_check(const cn_ctx* ctx, const cn_kvq4* c, int batch, int n_new) {
    CN_CHECK(ctx && c, CN_ERR_INVALID_ARG, "null argument");
    CN_CHECK(c->k_quants && c->k_scales && c->v_quants && c->v_scales, CN_ERR_INVALID_ARG, "null cache pointer");
    CN_CHECK(kvq4_head_dim_ok(c->head_dim), CN_ERR_UNSUPPORTED, "4-bit cache: head_dim %d (32, 64, 96, 128 or 256)",
             c->head_dim);
    CN_CHECK(c->n_seqs >= 1 && c->n_kv_heads >= 1 && c->ctx_len >= 1, CN_ERR_INVALID_ARG,
             "4-bit cache: bad shape (%d sequences, %d heads, %d positions)", c->n_seqs, c->n_kv_heads, c->ctx_len);
    CN_CHECK(c->ctx_len % 8 == 0, CN_ERR_INVALID_ARG, "4-bit cache: ctx_len %d is not a multiple of 8", c->ctx_len);
    const int64_t rows = (int64_t)c->n_kv_heads * c->ctx_len;
    CN_CHECK(c->seq_rows == 0 || (c->seq_rows >= rows && c->seq_rows % 8 == 0), CN_ERR_INVALID_ARG,
             "4-bit cache: seq_rows %lld is below %lld or not a multiple of 8", (long long)c->seq_rows,
             (long long)rows);
    // (byte offsets stay below 2^63)
    CN_CHECK(kvq4_seq_rows(*c) < (1ll << 40), CN_ERR_INVALID_ARG, "4-bit cache: seq_rows too large");
    const uintptr_t a = (uintptr_t)c->k_quants | (uintptr_t)c->k_scales | (uintptr_t)c->v_quants |
                        (uintptr_t)c->v_scales;
    CN_CHECK(a % 16 == 0, CN_ERR_INVALID_ARG, "4-bit cache: pointers must be 16-byte aligned");
    CN_CHECK(batch >= 1 && batch <= c->n_seqs, CN_ERR_INVALID_ARG, "batch %d outside [1, %d]", batch, c->n_seqs);
    CN_CHECK(n_new >= 1 && n_new <= c->ctx_len, CN_ERR_INVALID_ARG, "n_new %d outside [1, %d]", n_new, c->ctx_len);
    return CN_OK;
}

static int row_grid(const cn_kvq4& c, int batch, int n_new, int64_t* n_rows, dim3* grid) {
    *n_rows = (int64_t)batch * n_new * c.n_kv_heads;
    const int64_t ctas = (*n_rows + kRowThreads / 8 - 1) / (kRowThreads / 8);
    CN_CHECK(ctas < (1ll << 31), CN_ERR_INVALID_ARG, "too many rows (%lld)", (long long)*n_rows);
    *grid = dim3((unsigned)ctas, 2);
    return CN_OK;
}

#define KVQ4_BY_HD(hd, CALL) \
    switch (hd) {            \
        case 32: CALL(1);    \
        case 64: CALL(2);    \
        case 96: CALL(3);    \
        case 128: CALL(4);   \
        default: CALL(8);    \
    }

int kvq4_append(const cn_kvq4& c, const float* k, const float* v, int64_t kv_stride, const int* pos, const int* count,
                int batch, int n_new, const float2* rope, int neox, cudaStream_t st) {
    int64_t n;
    dim3 grid;
    int rc = row_grid(c, batch, n_new, &n, &grid);
    if (rc) return rc;
#define CALL(NB)                                                                                                 \
    kvq4_append_kernel<NB><<<grid, kRowThreads, 0, st>>>(                                                        \
        k, v, kv_stride, pos, count, n_new, c.n_kv_heads, n, rope, neox, static_cast<uint8_t*>(c.k_quants),      \
        static_cast<__half*>(c.k_scales), static_cast<uint8_t*>(c.v_quants), static_cast<__half*>(c.v_scales),   \
        kvq4_seq_rows(c), c.ctx_len);                                                                            \
    break
    KVQ4_BY_HD(c.head_dim, CALL)
#undef CALL
    CN_CUDA(cudaGetLastError());
    return CN_OK;
}

int kvq4_read(const cn_kvq4& c, float* k, float* v, int64_t kv_stride, const int* pos, const int* count, int batch,
              int n_new, cudaStream_t st) {
    int64_t n;
    dim3 grid;
    int rc = row_grid(c, batch, n_new, &n, &grid);
    if (rc) return rc;
#define CALL(NB)                                                                                                     \
    kvq4_read_kernel<NB><<<grid, kRowThreads, 0, st>>>(                                                              \
        k, v, kv_stride, pos, count, n_new, c.n_kv_heads, n, static_cast<const uint8_t*>(c.k_quants),                \
        static_cast<const __half*>(c.k_scales), static_cast<const uint8_t*>(c.v_quants),                             \
        static_cast<const __half*>(c.v_scales), kvq4_seq_rows(c), c.ctx_len);                                        \
    break
    KVQ4_BY_HD(c.head_dim, CALL)
#undef CALL
    CN_CUDA(cudaGetLastError());
    return CN_OK;
}

}  // namespace cn

using namespace cn;

extern "C" {

int cn_kvq4_append_dev(cn_ctx* ctx, const cn_kvq4* cache, const float* d_k, const float* d_v, int64_t kv_stride,
                       const int* d_pos, const int* d_count, int batch, int n_new, const float* d_rope, int rope_neox,
                       void* stream) {
    int rc = kvq4_check(ctx, cache, batch, n_new);
    if (rc) return rc;
    CN_CHECK(d_k && d_v && d_pos, CN_ERR_INVALID_ARG, "null argument");
    CN_CHECK(kv_stride >= (int64_t)cache->n_kv_heads * cache->head_dim, CN_ERR_INVALID_ARG,
             "kv_stride %lld is below %d values", (long long)kv_stride, cache->n_kv_heads * cache->head_dim);
    CN_CHECK(((uintptr_t)d_k | (uintptr_t)d_v) % 4 == 0 && (uintptr_t)d_rope % 8 == 0, CN_ERR_INVALID_ARG,
             "misaligned pointer");
    CN_CHECK(rope_neox == 0 || rope_neox == 1, CN_ERR_INVALID_ARG, "rope_neox is 0 or 1");
    DeviceScope ds(ctx->device);
    return kvq4_append(*cache, d_k, d_v, kv_stride, d_pos, d_count, batch, n_new,
                       reinterpret_cast<const float2*>(d_rope), rope_neox, (cudaStream_t)stream);
}

int cn_kvq4_read_dev(cn_ctx* ctx, const cn_kvq4* cache, float* d_k, float* d_v, int64_t kv_stride, const int* d_pos,
                     const int* d_count, int batch, int n_new, void* stream) {
    int rc = kvq4_check(ctx, cache, batch, n_new);
    if (rc) return rc;
    CN_CHECK((d_k || d_v) && d_pos, CN_ERR_INVALID_ARG, "null argument");
    CN_CHECK(kv_stride >= (int64_t)cache->n_kv_heads * cache->head_dim, CN_ERR_INVALID_ARG,
             "kv_stride %lld is below %d values", (long long)kv_stride, cache->n_kv_heads * cache->head_dim);
    CN_CHECK(((uintptr_t)d_k | (uintptr_t)d_v) % 4 == 0, CN_ERR_INVALID_ARG, "misaligned pointer");
    DeviceScope ds(ctx->device);
    return kvq4_read(*cache, d_k, d_v, kv_stride, d_pos, d_count, batch, n_new, (cudaStream_t)stream);
}

}  // extern "C"
