// kvq4.cuh -- the 4-bit KV cache: row layout, argument checks shared by its
// kernels (kvq4.cu: append and read; kvq4_attend.cu: attention).
//
// A row is the hd values of one (sequence, kv head, position), hd = 32 nb.
// Each block b of 32 values has an fp16 scale d and levels q in 0..15; a value
// is d * (q - 8).  Value e = 32 b + 8 i + g (i < 4, g < 8) is the nibble i & 1
// (low first) of byte g * 2 nb + 2 b + (i >> 1).  So chunk g (2 nb bytes)
// holds one value of every eighth dimension of all blocks, in 16-bit pieces
// per block: the tensor-core attention reads K as pairs of chunks (2t, 2t + 1)
// and V as single chunks, both straight in fragment order, with no shuffle
// and no table (see kvq4_attend.cu).
#pragma once

#include <math.h>

#include "cn_common.cuh"
#include "cn_internal.h"

namespace cn {

struct DeviceScope {  // the context's device for the length of a call
    int prev = -1;
    explicit DeviceScope(int dev) {
        cudaGetDevice(&prev);
        if (prev != dev) cudaSetDevice(dev);
        else prev = -1;
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

inline bool kvq4_head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

// Rows between two sequences' slots.
inline int64_t kvq4_seq_rows(const cn_kvq4& c) {
    return c.seq_rows ? c.seq_rows : (int64_t)c.n_kv_heads * c.ctx_len;
}

int kvq4_check(const cn_ctx* ctx, const cn_kvq4* c, int batch, int n_new);

// Enqueues (device set by the caller, arguments checked).
int kvq4_append(const cn_kvq4& c, const float* k, const float* v, int64_t kv_stride, const int* pos, const int* count,
                int batch, int n_new, const float2* rope, int neox, cudaStream_t st);
int kvq4_read(const cn_kvq4& c, float* k, float* v, int64_t kv_stride, const int* pos, const int* count, int batch,
              int n_new, cudaStream_t st);
int kvq4_attend(cn_ctx* ctx, const cn_kvq4& c, const float* q, int64_t q_stride, float* out, int64_t out_stride,
                const int* pos, const int* count, int batch, int n_new, int n_heads, float scale, const float2* rope,
                int neox, cudaStream_t st);

// The new tokens of sequence b that a call works on: tokens 0..n-1 at
// positions p0..p0+n-1; a negative position or count means none, and rows
// past the cache's end are left out.
__device__ __forceinline__ int kvq4_active(const int* pos, const int* count, int b, int n_new, int ctx_len, int& p0) {
    p0 = pos[b];
    int n = count ? min(count[b], n_new) : n_new;
    if (p0 < 0 || n <= 0 || p0 >= ctx_len) return 0;
    return min(n, ctx_len - p0);
}

}  // namespace cn
