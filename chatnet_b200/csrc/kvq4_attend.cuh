// kvq4_attend.cuh -- shared by the attention kernels over the 4-bit KV cache
// (kvq4_attend.cu: few rows; kvq4_prompt.cu: many).
#pragma once

#include <float.h>

#include "kvq4.cuh"

namespace cn {

struct AttendArgs {
    const float* q;
    float* out;
    int64_t q_stride, out_stride;
    const int* pos;
    const int* count;
    const float2* rope;
    const uint8_t *kq, *vq;
    const __half *kd, *vd;
    int64_t seq_rows;
    int batch, n_new, n_heads, n_kv, ctx_len, neox, groups;
    float mant;  // the scores' scale in log2 units, scale * log2(e) = mant * 2^exp, mant in [1/2, 1]
    int exp;
    uint32_t* err;
};

constexpr float kPeak = 9.f;  // the heaviest weight is 2^9 when a row's reference is set
constexpr float kLazy = 4.f;  // and the reference moves when a weight would pass 2^(9 + 4)

// What a row's sums count in log2 units, for queries times s * mant with s = 1 / inv
// a power of two: a power of two as well, so that sum * factor is exact and a
// score - R as exact as a subtraction, at any size.  Not 0 (-inf is a masked score), nor
// above 2^84: the sums lie below 2^43, so no score overflows, and scores that this takes
// down are still 0 or far more than a weight's whole range apart.
__device__ __forceinline__ float score_factor(float inv, int exp) {
    return fminf(fmaxf(scalbnf(inv, exp), FLT_MIN), 0x1p84f);
}
// The reference R for a maximum (a weight is 2^(score - R)); the maximum itself where
// scores are 16 apart and more, since one less 9 may come out as one less 16.
__device__ __forceinline__ float reference(float top) {
    const float r = top - kPeak;
    return top - r > 12.f ? top : r;
}

// Many rows: items of 128, head dimensions kvq4_prompt_ok.
bool kvq4_prompt_ok(int hd);
int kvq4_prompt_plan(cn_ctx* ctx, int64_t rows, int n_kv, int batch, int hd, int ctx_len, int* cluster, double* time);
int kvq4_attend_prompt(cn_ctx* ctx, int hd, int cluster, AttendArgs a, cudaStream_t st);

// mbar_wait as a short loop (the kernels wait in many places, and code beyond the
// instruction caches costs more than the waits).
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
#pragma unroll 1
    for (uint32_t i = 0; i < kSpinLimit; i++) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(addr), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

// D = A B + C on m16n8k16, free to be scheduled
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, const float* c) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// a b - c
__device__ __forceinline__ uint32_t h2_fms(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("{\n\t.reg .b32 n;\n\tneg.f16x2 n, %3;\n\tfma.rn.f16x2 %0, %1, %2, n;\n\t}" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// Nibbles 0 / 1 of both halves of x as level - 8, exactly (1024 + level, 1024 + 16 level).
__device__ __forceinline__ uint32_t even_levels(uint32_t x) {
    return h2_sub(lop3_and_or(x, 0x000F000Fu, 0x64006400u), 0x64086408u);
}
__device__ __forceinline__ uint32_t odd_levels(uint32_t x) {
    return h2_fma(lop3_and_or(x, 0x00F000F0u, 0x64006400u), 0x2C002C00u, 0xD480D480u);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(map_rank(addr, rank))
                 : "memory");
    return v;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_rank(addr, rank)) : "memory");
    return v;
}

// The halves of hi + lo = x: hi keeps 11 bits (x truncated, so the
// conversion is exact in fp16's normal range), lo the next 11.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float2 h = make_float2(__uint_as_float(__float_as_uint(a) & 0xFFFFE000u),
                                 __uint_as_float(__float_as_uint(b) & 0xFFFFE000u));
    const float2 l = fma2(h, make_float2(-1.f, -1.f), make_float2(a, b));
    hi = pack_half2(h.x, h.y);
    lo = pack_half2(l.x, l.y);
}

}  // namespace cn
