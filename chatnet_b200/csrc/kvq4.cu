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

constexpr int kRowThreads = 256;  // 8 lanes a row, 32 rows a CTA
constexpr float kMaxX = 524032.f;  // 8 * 65504

__device__ __forceinline__ float tame(float x) {
    return x == x ? fminf(fmaxf(x, -kMaxX), kMaxX) : 0.f;
}

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: whole numbers from here on

// The nearest level to x / d, halves up, in the low 16 bits, for any d.  x times
// the rounded 1 / d, rounded to a whole number q, is off by one at most; the rest
// x - d q is exact in fp32 there (both terms lie within a factor of two, or q is
// 0) and decides against half a step.
__device__ __noinline__ uint32_t level_exact(float x, float d, float inv) {
    const float f = fmaf(x, inv, kWhole + 8.f), q = f - (kWhole + 8.f);
    const float rest = __uint_as_float(__float_as_uint(fmaf(-d, q, x)) ^ (__float_as_uint(d) & 0x80000000u));
    const float half = 0.5f * fabsf(d);
    int n = __float_as_int(f);
    if (rest >= half) n++;
    if (rest < -half) n--;
    const int zero = __float_as_int(kWhole);
    return (uint32_t)min(max(n, zero), zero + 15);
}
// The same away from the borders: `near` is set where x / d (known to 2^-21) may
// be within 10^-5 of one.  d is at least 2^-14, so that x / d is above -8.01.
__device__ __forceinline__ uint32_t level(float x, float inv, bool& near) {
    const float f = fmaf(x, inv, kWhole + 8.f), q = f - (kWhole + 8.f);
    near |= fabsf(fmaf(x, inv, -q)) > 0.49999f;
    return (uint32_t)min(__float_as_int(f), __float_as_int(kWhole) + 15);
}

// Which row a thread's eight lanes take.  Many tokens: a CTA has 32 tokens of one
// head of one sequence (their rows are neighbours in the cache), from the block's
// indexes alone.  Few: rows side by side, heads first.
struct RowAt {
    int b, i, h;
    bool in;
    __device__ RowAt(uint32_t n_rows, int n_new, int n_kv, bool many) {
        if (many) {
            i = blockIdx.x * 32 + (threadIdx.x >> 3);
            h = blockIdx.y >> 1;
            b = blockIdx.z;
            in = i < n_new;
        } else {
            const uint32_t r = blockIdx.x * 32 + (threadIdx.x >> 3), t = r / (uint32_t)n_kv;
            h = (int)(r % (uint32_t)n_kv);
            b = (int)(t / (uint32_t)n_new);
            i = (int)(t % (uint32_t)n_new);
            in = r < n_rows;
        }
    }
};

}  // namespace

// Eight lanes a row, so that a block's minimum and maximum need three shuffles
// for four rows at once.  Lane l holds the values 4l .. 4l + 3 of every block (16-byte
// loads and stores): the nibbles i = l >> 1 of chunks g = 4 (l & 1) .. + 3.  A
// word holds two 16-bit pieces; the four lanes of one parity OR their nibbles
// together, and lane l then writes chunk 4 (l & 1) + (l >> 1).  The fp32 rows'
// bytes would bound it (48 us for the case below); with about 500 instructions per 16
// values for rotation, scale, levels and packing, issue does (80 % of the slots; without
// the rotation 76 us).  8191 tokens of 32 heads of 128: 80 us, 3.9 TB/s; followed by
// reading them back 132, and 149 with rows side by side for many tokens too and the
// exact level for every value.
template <int NB>
__global__ void __launch_bounds__(kRowThreads)
    kvq4_append_kernel(const float* __restrict__ k, const float* __restrict__ v, int64_t kv_stride,
                       const int* __restrict__ pos, const int* __restrict__ count, int n_new, int n_kv,
                       uint32_t n_rows, const float2* __restrict__ rope, int neox, uint8_t* __restrict__ kq,
                       __half* __restrict__ kd, uint8_t* __restrict__ vq, __half* __restrict__ vd, int64_t seq_rows,
                       int ctx_len, int wide, int many) {
    constexpr int HD = 32 * NB, H = HD / 2;
    const int l = threadIdx.x & 7;
    const RowAt at(n_rows, n_new, n_kv, many);
    const bool is_v = blockIdx.y & 1;
    bool live = at.in && (is_v ? v : k) != nullptr;
    int64_t tok = 0, dst = 0;
    const int h = at.h;
    int p = 0;
    if (live) {
        tok = (int64_t)at.b * n_new + at.i;
        int p0;
        live = at.i < kvq4_active(pos, count, at.b, n_new, ctx_len, p0);
        p = p0 + at.i;
        dst = (int64_t)at.b * seq_rows + (int64_t)h * ctx_len + p;
    }
    float4 x[NB];
    const float* src = (is_v ? v : k) + tok * kv_stride + (int64_t)h * HD;
    auto get = [&](int e) {  // (rows that are not 16-byte aligned: value by value)
        return wide ? *reinterpret_cast<const float4*>(src + e)
                    : make_float4(src[e], src[e + 1], src[e + 2], src[e + 3]);
    };
#pragma unroll
    for (int b = 0; b < NB; b++) x[b] = live ? get(32 * b + 4 * l) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (!is_v && rope && live) {
        const float2* tab = rope + (int64_t)p * H;
        auto lo = [](float a, float c, float2 cs) { return __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(c, cs.y)); };
        auto hi = [](float a, float c, float2 cs) { return __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(c, cs.x)); };
        if (!neox) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float4 cs = *reinterpret_cast<const float4*>(tab + 16 * b + 2 * l);
                const float2 c0 = {cs.x, cs.y}, c1 = {cs.z, cs.w};
                const float4 y = x[b];
                x[b] = make_float4(lo(y.x, y.y, c0), hi(y.x, y.y, c0), lo(y.z, y.w, c1), hi(y.z, y.w, c1));
            }
        } else if constexpr (NB % 2 == 0) {  // e pairs with e + hd/2: the same lane holds both
#pragma unroll
            for (int b = 0; b < NB / 2; b++) {
                const float4* cs = reinterpret_cast<const float4*>(tab + 32 * b + 4 * l);
                const float4 s0 = cs[0], s1 = cs[1];
                const float2 c0 = {s0.x, s0.y}, c1 = {s0.z, s0.w}, c2 = {s1.x, s1.y}, c3 = {s1.z, s1.w};
                const float4 y = x[b], z = x[b + NB / 2];
                x[b] = make_float4(lo(y.x, z.x, c0), lo(y.y, z.y, c1), lo(y.z, z.z, c2), lo(y.w, z.w, c3));
                x[b + NB / 2] = make_float4(hi(y.x, z.x, c0), hi(y.y, z.y, c1), hi(y.z, z.z, c2), hi(y.w, z.w, c3));
            }
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int e = 32 * b + 4 * l;
                const bool first = e < H;
                const float4 y = x[b], z = get(first ? e + H : e - H);
                const float2* cs = tab + (first ? e : e - H);
                const float2 c0 = cs[0], c1 = cs[1], c2 = cs[2], c3 = cs[3];
                x[b] = first ? make_float4(lo(y.x, z.x, c0), lo(y.y, z.y, c1), lo(y.z, z.z, c2), lo(y.w, z.w, c3))
                             : make_float4(hi(z.x, y.x, c0), hi(z.y, y.y, c1), hi(z.z, y.z, c2), hi(z.w, y.w, c3));
            }
        }
    }
    uint32_t piece[NB];  // of chunk 4 (l & 1) + (l >> 1)
    float scale = 0.f;   // of block l
    const int nib = 4 * (l >> 1);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float4 y = x[b];
        float lo = min_nan(min_nan(y.x, y.y), min_nan(y.z, y.w)), hi = max_nan(max_nan(y.x, y.y), max_nan(y.z, y.w));
        if (!(lo >= -kMaxX && hi <= kMaxX)) {  // (rarely)
            y = make_float4(tame(y.x), tame(y.y), tame(y.z), tame(y.w));
            lo = fminf(fminf(y.x, y.y), fminf(y.z, y.w));
            hi = fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w));
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const float d = __half2float(__float2half_rn(__fmul_rn(-lo >= hi ? lo : hi, -0.125f)));
        uint32_t w0 = 0x00080008u << nib, w1 = w0;  // level 8: the value 0
        if (d != 0.f) {
            const float inv = __frcp_rn(d);
            bool near = fabsf(d) < 6.103515625e-5f;
            uint32_t q0 = level(y.x, inv, near), q1 = level(y.y, inv, near), q2 = level(y.z, inv, near),
                     q3 = level(y.w, inv, near);
            if (near) {
                q0 = level_exact(y.x, d, inv), q1 = level_exact(y.y, d, inv), q2 = level_exact(y.z, d, inv),
                q3 = level_exact(y.w, d, inv);
            }
            w0 = __byte_perm(q0, q1, 0x5410) << nib;
            w1 = __byte_perm(q2, q3, 0x5410) << nib;
        }
#pragma unroll
        for (int o = 2; o <= 4; o <<= 1) {
            w0 |= __shfl_xor_sync(0xffffffffu, w0, o);
            w1 |= __shfl_xor_sync(0xffffffffu, w1, o);
        }
        const uint32_t w = (l >> 2) ? w1 : w0;
        piece[b] = (l & 2) ? w >> 16 : w & 0xFFFFu;
        if (l == b) scale = d;
    }
    if (!live) return;
    uint8_t* q = (is_v ? vq : kq) + dst * (HD / 2) + (4 * (l & 1) + (l >> 1)) * (2 * NB);
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
    if (l < NB) ((is_v ? vd : kd) + dst * NB)[l] = __float2half_rn(scale);
}

// Eight lanes a row, lane l the values 4l .. 4l + 3 of every block.  Bound by the bytes,
// most of them written: 8191 tokens of 32 heads of 128 take 61 us, 5.0 TB/s.
template <int NB>
__global__ void __launch_bounds__(kRowThreads)
    kvq4_read_kernel(float* __restrict__ k, float* __restrict__ v, int64_t kv_stride, const int* __restrict__ pos,
                     const int* __restrict__ count, int n_new, int n_kv, uint32_t n_rows,
                     const uint8_t* __restrict__ kq,
                     const __half* __restrict__ kd, const uint8_t* __restrict__ vq, const __half* __restrict__ vd,
                     int64_t seq_rows, int ctx_len, int wide, int many) {
    constexpr int HD = 32 * NB;
    const int l = threadIdx.x & 7;
    const RowAt at(n_rows, n_new, n_kv, many);
    const bool is_v = blockIdx.y & 1;
    float* out = is_v ? v : k;
    if (!at.in || !out) return;
    int p0;
    if (at.i >= kvq4_active(pos, count, at.b, n_new, ctx_len, p0)) return;
    const int h = at.h;
    const int64_t tok = (int64_t)at.b * n_new + at.i;
    const int64_t src = (int64_t)at.b * seq_rows + (int64_t)h * ctx_len + p0 + at.i;
    // chunks 4 (l & 1) .. + 3 of the row, 4 NB pieces
    uint32_t w[2 * NB];
    const uint8_t* q = (is_v ? vq : kq) + src * (HD / 2) + (l & 1) * (8 * NB);
    if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int j = 0; j < NB / 2; j++) {
            const uint4 u = reinterpret_cast<const uint4*>(q)[j];
            w[4 * j] = u.x, w[4 * j + 1] = u.y, w[4 * j + 2] = u.z, w[4 * j + 3] = u.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 2 * NB; j++) w[j] = reinterpret_cast<const uint32_t*>(q)[j];
    }
    const __half* d = (is_v ? vd : kd) + src * NB;
    out += tok * kv_stride + (int64_t)h * HD + 4 * l;
    const int nib = 4 * (l >> 1);
#pragma unroll
    for (int bl = 0; bl < NB; bl++) {
        const float s = __half2float(d[bl]);
        float x[4];
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int piece = g * NB + bl;
            x[g] = s * (float)((int)((w[piece / 2] >> (16 * (piece % 2) + nib)) & 15u) - 8);
        }
        if (wide) {
            *reinterpret_cast<float4*>(out + 32 * bl) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int g = 0; g < 4; g++) out[32 * bl + g] = x[g];
        }
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
    // (the end of the last tile, and of what a cluster steps past it, stays below 2^31)
    CN_CHECK(c->ctx_len <= 1 << 30, CN_ERR_INVALID_ARG, "4-bit cache: ctx_len %d is above 2^30", c->ctx_len);
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

static int row_grid(const cn_kvq4& c, int batch, int n_new, uint32_t* n_rows, int* many, dim3* grid) {
    const int64_t n = (int64_t)batch * n_new * c.n_kv_heads;
    CN_CHECK(n < (1ll << 31), CN_ERR_INVALID_ARG, "too many rows (%lld)", (long long)n);
    *n_rows = (uint32_t)n;
    *many = n_new >= 16 && batch <= 65535 && c.n_kv_heads <= 32767;
    *grid = *many ? dim3((unsigned)((n_new + 31) / 32), 2 * (unsigned)c.n_kv_heads, (unsigned)batch)
                  : dim3((unsigned)((n + 31) / 32), 2);
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
    uint32_t n;
    int many;
    dim3 grid;
    int rc = row_grid(c, batch, n_new, &n, &many, &grid);
    if (rc) return rc;
    const int wide = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && kv_stride % 4 == 0;
#define CALL(NB)                                                                                                 \
    kvq4_append_kernel<NB><<<grid, kRowThreads, 0, st>>>(                                                        \
        k, v, kv_stride, pos, count, n_new, c.n_kv_heads, n, rope, neox, static_cast<uint8_t*>(c.k_quants),      \
        static_cast<__half*>(c.k_scales), static_cast<uint8_t*>(c.v_quants), static_cast<__half*>(c.v_scales),   \
        kvq4_seq_rows(c), c.ctx_len, wide, many);                                                                            \
    break
    KVQ4_BY_HD(c.head_dim, CALL)
#undef CALL
    CN_CUDA(cudaGetLastError());
    return CN_OK;
}

int kvq4_read(const cn_kvq4& c, float* k, float* v, int64_t kv_stride, const int* pos, const int* count, int batch,
              int n_new, cudaStream_t st) {
    uint32_t n;
    int many;
    dim3 grid;
    int rc = row_grid(c, batch, n_new, &n, &many, &grid);
    if (rc) return rc;
    const int wide = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && kv_stride % 4 == 0;
#define CALL(NB)                                                                                                     \
    kvq4_read_kernel<NB><<<grid, kRowThreads, 0, st>>>(                                                              \
        k, v, kv_stride, pos, count, n_new, c.n_kv_heads, n, static_cast<const uint8_t*>(c.k_quants),                \
        static_cast<const __half*>(c.k_scales), static_cast<const uint8_t*>(c.v_quants),                             \
        static_cast<const __half*>(c.v_scales), kvq4_seq_rows(c), c.ctx_len, wide, many);                                  \
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
    CN_CHECK(((uintptr_t)d_k | (uintptr_t)d_v) % 4 == 0 && (uintptr_t)d_rope % 16 == 0, CN_ERR_INVALID_ARG,
             "misaligned pointer (k and v 4 bytes, the rope table 16)");
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
