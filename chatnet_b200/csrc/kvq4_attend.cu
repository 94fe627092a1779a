// kvq4_attend.cu -- attention over the 4-bit KV cache (cn_kvq4_attend_dev).
//
//   o = sum_p w_p v_p / sum_p w_p,  w_p = exp(scale (q . k_p) - max)
// over positions p = 0 .. pos[b] + i of token i, with one pass over the cache
// (running maximum and sum, fp32).
//
// Rows: the queries that read one kv head of one sequence, row r = token
// r / mul, query head kvh * mul + r % mul (mul = n_heads / n_kv).
#include <float.h>
#include <math.h>

#include "kvq4.cuh"
#include "kvq4_attend.cuh"

namespace cn {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxCluster = 16;

// positions of a warp's tile, bytes of a tile in the ring (quants and scales of K and V)
__host__ __device__ constexpr int tile_pos(int nb) { return nb <= 4 ? 48 : 32; }
__host__ __device__ constexpr int tile_bytes(int nb) { return tile_pos(nb) * 36 * nb; }
constexpr int kRing = 2;  // tiles in a warp's ring
// a tile's scales laid out for the fragments (K's as fp32, then V's as fp16), per warp
__host__ __device__ constexpr int scale_bytes(int nb) { return tile_pos(nb) * 4 * nb; }
// the rows' query fragments
__host__ __device__ constexpr int query_bytes(int nb) { return 32 * 32 * nb; }
__host__ __device__ constexpr int ctas_per_sm(int nb) { return nb <= 4 ? 3 : 2; }

// Rotated query values e, e + 1 (e even) of one row.
template <int HD>
__device__ __forceinline__ float2 query_pair(const float* __restrict__ x, const float2* __restrict__ tab, int neox,
                                             int e) {
    const float2 a = *reinterpret_cast<const float2*>(x + e);
    if (!tab) return a;
    if (!neox) {
        const float2 cs = tab[e / 2];
        return make_float2(__fsub_rn(__fmul_rn(a.x, cs.x), __fmul_rn(a.y, cs.y)),
                           __fadd_rn(__fmul_rn(a.x, cs.y), __fmul_rn(a.y, cs.x)));
    }
    constexpr int H = HD / 2;
    const bool first = e < H;
    const float2 b = *reinterpret_cast<const float2*>(x + (first ? e + H : e - H));
    const float4 cs = *reinterpret_cast<const float4*>(tab + (first ? e : e - H));
    if (first)
        return make_float2(__fsub_rn(__fmul_rn(a.x, cs.x), __fmul_rn(b.x, cs.y)),
                           __fsub_rn(__fmul_rn(a.y, cs.z), __fmul_rn(b.y, cs.w)));
    return make_float2(__fadd_rn(__fmul_rn(b.x, cs.y), __fmul_rn(a.x, cs.x)),
                       __fadd_rn(__fmul_rn(b.y, cs.w), __fmul_rn(a.y, cs.z)));
}

// N 32-bit (or 16-bit) words from shared memory with the widest loads the
// row layout allows.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t* w, const uint8_t* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}
// NB 16-bit values: two per word
template <int NB>
__device__ __forceinline__ void lds_halves(uint32_t* w, const uint8_t* p) {
    if constexpr (NB % 2 == 0) {
        lds_words<NB / 2>(w, p);
    } else {
#pragma unroll
        for (int i = 0; i < NB; i += 2)
            w[i / 2] = (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] |
                       (i + 1 < NB ? (uint32_t) reinterpret_cast<const uint16_t*>(p)[i + 1] << 16 : 0u);
    }
}
__device__ __forceinline__ float half_at(const uint32_t* w, int b) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w[b >> 1]);
    return (b & 1) ? __high2float(h) : __low2float(h);
}
// {16-bit piece i of a, piece j of b}
__device__ __forceinline__ uint32_t pair16(const uint32_t* a, int i, const uint32_t* b, int j) {
    return __byte_perm(a[i >> 1], b[j >> 1], ((i & 1) ? 0x32u : 0x10u) | ((j & 1) ? 0x7600u : 0x5400u));
}

}  // namespace

// Few rows against a long cache (decode).  An item is eight rows of one
// (sequence, kv head); its CTAs form a cluster, and every warp of it takes
// its share of the tiles of 48 positions through a ring of bulk copies of its own,
// with its own running reference, sum and output.  The partials meet in shared
// memory, first the CTA's, then the cluster's: no workspace, no atomics, one
// launch.
//
// Scores: S = Q K^T on mma.m16n8k16, the eight rows' high halves in the
// tile's rows 0-7 and their low halves in rows 8-15 (q scaled to [2^13, 2^15]
// as for score_factor, each entry's halves with 11 bits of its own, so that small
// entries next to a large one keep 22 too).  K's levels go in signed, exact in fp16,
// two instructions for two values: as the bare nibbles they would take one, but then
// -8 sum(q) has to be taken off again, whose rounding drowns the small entries beside
// a large one.  The block's scale multiplies the block's sum in fp32.
// Output: O = W V with V's signed levels exact in fp16 and w_p d_p,b (weight
// times the block's scale) as two halves: w's halves hi, lo times the fp16 d
// give h = hi d rounded, then its exact rounding error and lo d in the second
// half, all in packed fp16 (three instructions for two positions).  A row's
// weights are 2^9 at its reference (a running maximum in log2 units, moved when
// outgrown by 2^4), and V's scales count 2^e times where the largest seen
// lies outside [2^-7, 4), so w d stays below 2^15 and keeps 22 bits down to 2^-25
// of that, whatever the cache's range.  Each tile's products are summed from
// zero and joined in fp32 (the tensor cores truncate where fp32 rounds).
//
// Bound: latency.  168 registers a thread let three CTAs on an SM, and its twelve warps
// (ten active) wait for one MMA's or conversion's result after the other: at 32 thousand
// positions 46 % of the issue slots are used and 31 % of DRAM's rate (the loads alone run
// at the copy rate).  Short sequences pay each CTA's set-up, first loads and two merges
// besides (16 at 2047: 31 % of the slots), and with one query head to a kv head 14 of the
// 16 rows of every MMA are empty.  8 sequences of 131 thousand positions, 64 heads over 8
// of 128: 314 us, 3.0 TB/s; 16 to 2047: 19.3 us; 32 to 1001, 32 kv heads: 57 us, 2 TB/s;
// one of 512, 4 kv heads of 64: 6.2 us.
template <int NB>
__global__ void __launch_bounds__(32 * kWarps, ctas_per_sm(NB)) kvq4_attend_rows_kernel(const AttendArgs a) {
    constexpr int HD = 32 * NB, RB = 16 * NB, SB = 2 * NB;  // bytes of a row's quants and scales
    constexpr int TP = tile_pos(NB), TB = tile_bytes(NB), NT = TP / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kWarps][kRing];
    __shared__ float sR[kWarps + 1][8], sL[kWarps + 1][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t cs = cluster_size(), rank = cluster_rank();
    const int item = (int)(blockIdx.x / cs);
    const int grp = item % a.groups, bh = item / a.groups, kvh = bh % a.n_kv;
    int b = bh / a.n_kv;
    if (a.batch > 1 && a.batch <= 32) {
        // the longest sequences first: what starts last is short
        const int mine = lane < a.batch ? a.pos[lane] : -1;
        int before = 0;
        for (int k = 0; k < a.batch; k++) {
            const int other = __shfl_sync(0xffffffffu, mine, k);
            before += other > mine || (other == mine && k < lane);
        }
        b = __ffs(__ballot_sync(0xffffffffu, lane < a.batch && before == b)) - 1;
    }
    const int mul = a.n_heads / a.n_kv;
    int p0;
    const int n = kvq4_active(a.pos, a.count, b, a.n_new, a.ctx_len, p0);
    const int rows = n * mul - 8 * grp;  // of this item (more than 8: 8)
    if (rows <= 0) return;               // (the whole cluster)
    const int r0 = 8 * grp;
    const int len = p0 + min(n - 1, (r0 + 7) / mul) + 1;  // positions any of the rows sees
    const int tiles = (len + TP - 1) / TP, step = (int)cs * kWarps;  // this warp's: tile0, tile0 + step, ...
    const int tile0 = (int)rank * kWarps + warp;
    const int64_t base = (int64_t)b * a.seq_rows + (int64_t)kvh * a.ctx_len;
    uint8_t* ring = smem + warp * kRing * TB;
    float* fs = reinterpret_cast<float*>(smem + kWarps * kRing * TB + warp * scale_bytes(NB));
    uint4* qs = reinterpret_cast<uint4*>(smem + kWarps * (kRing * TB + scale_bytes(NB)));  // [2 NB][32]

    auto issue = [&](int tile, int s) {  // one lane
        const int64_t row = base + (int64_t)tile * TP;
        const int np = min(TP, (len - tile * TP + 7) & ~7);  // (ctx_len is a multiple of 8)
        uint8_t* d = ring + s * TB;
        uint64_t* bar = &full[warp][s];
        mbar_expect_tx(bar, (uint32_t)(np * 36 * NB));
        bulk_load(d, a.kq + row * RB, np * RB, bar);
        bulk_load(d + TP * RB, a.vq + row * RB, np * RB, bar);
        bulk_load(d + 2 * TP * RB, a.kd + row * NB, np * SB, bar);
        bulk_load(d + 2 * TP * RB + TP * SB, a.vd + row * NB, np * SB, bar);
    };
    if (lane == 0) {
        for (int s = 0; s < kRing; s++) mbar_init(&full[warp][s], 1);
        fence_mbar_init();
        fence_proxy_async();
        for (int s = 0; s < kRing; s++)
            if (tile0 + s * step < tiles) issue(tile0 + s * step, s);
    }

    // the rows' queries as A fragments in shared memory (every warp needs a
    // row's maximum, block j is left by warp j % kWarps); limit = last position
    // the row sees
    float factor;
    int limit;
    {
        const int r = r0 + min(g, rows - 1);
        const int tok = r / mul;
        limit = p0 + tok;
        const float* x = a.q + ((int64_t)b * a.n_new + tok) * a.q_stride + (int64_t)(kvh * mul + r % mul) * HD;
        const float2* tab = a.rope ? a.rope + (int64_t)limit * (HD / 2) : nullptr;
        float2 v[NB][4];
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[j][i] = query_pair<HD>(x, tab, a.neox, 32 * j + 8 * i + 2 * t);
                amax = fmaxf(amax, fmaxf(fabsf(v[j][i].x), fabsf(v[j][i].y)));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        float sc, inv;
        row_pow2_scale(amax, sc, inv);
        factor = score_factor(inv, a.exp);
        sc *= a.mant;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            if (j % kWarps != warp) continue;
            uint32_t qa[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x0 = v[j][i].x * sc, x1 = v[j][i].y * sc;
                const uint32_t hi = pack_half2(x0, x1);
                const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                // a0 / a1: high and low halves of k 2t, 2t+1; a2 / a3: of k 2t+8, 2t+9
                qa[4 * (i >> 1) + 2 * (i & 1)] = hi;
                qa[4 * (i >> 1) + 2 * (i & 1) + 1] = pack_half2(x0 - hf.x, x1 - hf.y);
            }
            qs[64 * j + lane] = make_uint4(qa[0], qa[1], qa[2], qa[3]);
            qs[64 * j + 32 + lane] = make_uint4(qa[4], qa[5], qa[6], qa[7]);
        }
    }

    float2 o[4 * NB];
#pragma unroll
    for (int j = 0; j < 4 * NB; j++) o[j] = make_float2(0.f, 0.f);
    float R = -FLT_MAX;
    float2 l2 = make_float2(0.f, 0.f);
    uint32_t dtop = 0;  // bound of the |V scale| seen, fp16 bits
    int e2 = 0;         // V's scales count 2^e2 times
    bool ok = true, fresh = true;
    const int seen_by_all = p0 + r0 / mul + 1;  // positions every row sees
    // column c of a score tile is position c ^ ((c >> 1) & 1) of its eight: rows
    // of both parities for the four t of a V load, and for K's
    const int kcol = g ^ ((g >> 1) & 1);
    const int c0 = (2 * t) ^ (t & 1), c1 = (2 * t + 1) ^ (t & 1);
    // where position `lane` of 32 goes among the pairs of columns: 2 * (4 * (tile of 8) + t) + (column & 1)
    const int mypair = (lane & 24) | ((lane & 7) ^ ((lane >> 1) & 1));
    __syncthreads();  // the queries
    int s = 0;
    uint32_t parity = 0;
    for (int tile = tile0; tile < tiles; tile += step) {
        if (ok && !bar_wait(&full[warp][s], parity)) {
            ok = false;
            if (lane == 0) atomicOr(a.err, kErrTimeout);
            bar_wait(&full[warp][s ^ 1], parity ^ s);  // (nor does the other copy outlive the CTA, if there is one)
            bar_wait(&full[warp][s], parity);
        }
        const uint8_t* sk = ring + s * TB;
        const uint8_t* sv = sk + TP * RB;
        const uint8_t* skd = sv + TP * RB;
        const uint8_t* svd = skd + TP * SB;
        const int first = tile * TP;

        // ---- scores ----
        // K's scales as fp32, the two columns of a thread side by side
#pragma unroll
        for (int k = 0; k < TP; k += 32) {
            if (k + 32 > TP && lane >= TP - k) break;
            uint32_t h[(NB + 1) / 2];
            lds_halves<NB>(h, skd + (k + lane) * SB);
#pragma unroll
            for (int j = 0; j < NB; j++) fs[(k / 2 + (mypair >> 1)) * 2 * NB + 2 * j + (mypair & 1)] = half_at(h, j);
        }
        __syncwarp();
        float2 p[NT];
        {
            uint32_t w[NT][NB];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                lds_words<NB>(w[nt], sk + (8 * nt + kcol) * RB + t * 4 * NB);
                p[nt] = make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const uint4 qa = qs[64 * j + lane], qb = qs[64 * j + 32 + lane];
                const uint32_t a0[4] = {qa.x, qa.y, qa.z, qa.w}, a1[4] = {qb.x, qb.y, qb.z, qb.w};
                float c[NT][4];
                uint32_t y[NT];
                // (the tiles side by side: an MMA's result is long in coming)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const uint32_t x = pair16(w[nt], j, w[nt], NB + j);
                    c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
                    mma(c[nt], a0, even_levels(x), odd_levels(x), c[nt]);
                    y[nt] = x >> 8;
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma(c[nt], a1, even_levels(y[nt]), odd_levels(y[nt]), c[nt]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float2 d = reinterpret_cast<const float2*>(fs)[(4 * nt + t) * NB + j];
                    p[nt] = fma2(d, add2(make_float2(c[nt][0], c[nt][1]), make_float2(c[nt][2], c[nt][3])), p[nt]);
                }
            }
        }
        float top = -INFINITY;
        if (first + TP > seen_by_all) {  // positions some row does not see
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if (first + 8 * nt + c0 > limit) p[nt].x = -INFINITY;
                if (first + 8 * nt + c1 > limit) p[nt].y = -INFINITY;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) top = fmaxf(top, fmaxf(p[nt].x, p[nt].y));
        top *= factor;

        // ---- reference, and V's scales ----
        {
            constexpr int K = (TP + 31) / 32;
            uint32_t h[K][(NB + 1) / 2], mx = 0;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int q = 32 * k + lane;
                const bool in = (32 * k + 32 <= TP || q < TP) && first + q < len;  // (rows past the end hold anything)
                lds_halves<NB>(h[k], svd + (in ? q : 0) * SB);
#pragma unroll
                for (int j = 0; j < (NB + 1) / 2; j++) {
                    if (!in) h[k][j] = 0;
                    mx = __vmaxu2(mx, h[k][j] & 0x7FFF7FFFu);
                }
            }
            mx = max(mx & 0xFFFFu, mx >> 16);
            if (__any_sync(0xffffffffu, top - R > kPeak + kLazy || mx > dtop)) {
                float grow = 1.f;
                mx = __reduce_max_sync(0xffffffffu, mx);
                if (mx > dtop) {
                    // the scales lie below 2^E
                    dtop = mx | 0x3FFu;
                    const int E = (int)(dtop >> 10) - 14, ne = E >= -6 && E <= 2 ? 0 : min(2 - E, 15);
                    grow = fresh ? 1.f : exp2f((float)(ne - e2));
                    e2 = ne;
                    fresh = false;
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                float al = 1.f;
                if (top - R > kPeak + kLazy) {
                    const float to = reference(top);
                    al = ex2(R - to);
                    R = to;
                }
                l2.x *= al;
                l2.y *= al;
                al *= grow;
#pragma unroll
                for (int j = 0; j < 4 * NB; j++) {
                    o[j].x *= al;
                    o[j].y *= al;
                }
            }
            const uint32_t f = (uint32_t)(15 + e2) * 0x04000400u;  // 2^e2 (-14..15), twice
            __syncwarp();  // (K's are read)
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (32 * k + 32 > TP && lane >= TP - 32 * k) break;
#pragma unroll
                for (int j = 0; j < NB; j += 2) {
                    const uint32_t v = h2_mul(h[k][j / 2], f);
                    uint16_t* q = reinterpret_cast<uint16_t*>(fs) + ((16 * k + (mypair >> 1)) * NB + j) * 2 + (mypair & 1);
                    q[0] = (uint16_t)v;
                    if (j + 1 < NB) q[2] = (uint16_t)(v >> 16);
                }
            }
            __syncwarp();
        }

        // ---- output ----
        uint32_t hi[NT], lo[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            p[nt].x = ex2(fmaf(p[nt].x, factor, -R));
            p[nt].y = ex2(fmaf(p[nt].y, factor, -R));
            l2 = add2(l2, p[nt]);
            split2(p[nt].x, p[nt].y, hi[nt], lo[nt]);
        }
#pragma unroll
        for (int jp = 0; jp < NB; jp += 2) {  // two blocks: one word of a chunk
            float c[2][4][4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                c[0][i][0] = c[0][i][1] = c[0][i][2] = c[0][i][3] = c[1][i][0] = c[1][i][1] = c[1][i][2] = c[1][i][3] = 0.f;
#pragma unroll
            for (int k = 0; k < NT / 2; k++) {
                uint32_t w[4], d[2][2];
#pragma unroll
                for (int n2 = 0; n2 < 2; n2++) {
                    const int nt = 2 * k + n2;
                    const uint32_t* dp = reinterpret_cast<const uint32_t*>(fs) + (4 * nt + t) * NB + jp;
                    if constexpr (NB % 2 == 0) {
                        const uint2 v = *reinterpret_cast<const uint2*>(dp);
                        d[0][n2] = v.x;
                        d[1][n2] = v.y;
                    } else {
                        d[0][n2] = dp[0];
                        d[1][n2] = jp + 1 < NB ? dp[1] : 0u;
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint8_t* wp = sv + (8 * nt + (u ? c1 : c0)) * RB + g * 2 * NB + 2 * jp;
                        if constexpr (NB % 2 == 0)
                            w[2 * n2 + u] = *reinterpret_cast<const uint32_t*>(wp);
                        else
                            w[2 * n2 + u] =
                                (uint32_t) * reinterpret_cast<const uint16_t*>(wp) |
                                (jp + 1 < NB ? (uint32_t) reinterpret_cast<const uint16_t*>(wp)[1] << 16 : 0u);
                    }
                }
#pragma unroll
                for (int jj = 0; jj < 2; jj++) {
                    if (jp + jj >= NB) break;
                    uint32_t af[4], x0, x1;
#pragma unroll
                    for (int n2 = 0; n2 < 2; n2++) {
                        const uint32_t dd = d[jj][n2], h = h2_mul(hi[2 * k + n2], dd);
                        af[2 * n2] = h;
                        af[2 * n2 + 1] = h2_fma(lo[2 * k + n2], dd, h2_fms(hi[2 * k + n2], dd, h));
                    }
                    x0 = pair16(w, jj, w + 1, jj);
                    x1 = pair16(w + 2, jj, w + 3, jj);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (i & 1) mma(c[jj][i], af, odd_levels(x0), odd_levels(x1), c[jj][i]);
                        else mma(c[jj][i], af, even_levels(x0), even_levels(x1), c[jj][i]);
                        if (i == 1) {
                            x0 >>= 8;
                            x1 >>= 8;
                        }
                    }
                }
            }
#pragma unroll
            for (int jj = 0; jj < 2; jj++) {
                if (jp + jj >= NB) break;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float* f = c[jj][i];
                    float2& r = o[4 * (jp + jj) + i];
                    r = add2(r, add2(make_float2(f[0], f[1]), make_float2(f[2], f[3])));
                }
            }
        }
        __syncwarp();
        if (lane == 0 && ok && tile + kRing * step < tiles) issue(tile + kRing * step, s);
        if (++s == kRing) {
            s = 0;
            parity ^= 1;
        }
    }

    // ---- the CTA's partials, then the cluster's ----
    float l = l2.x + l2.y;
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    __syncthreads();  // every warp is done with its ring
    float* so = reinterpret_cast<float*>(smem);  // [kWarps + 1][8][HD]: the warps', then the CTA's
    const float un = exp2f((float)-e2);
    if (t == 0) {
        sR[warp][g] = R;
        sL[warp][g] = l;
    }
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<float2*>(so + (warp * 8 + g) * HD + 32 * j + 8 * i + 2 * t) =
                make_float2(o[4 * j + i].x * un, o[4 * j + i].y * un);
    __syncthreads();
    float* sc = so + kWarps * 8 * HD;
    for (int e = threadIdx.x; e < 8 * HD / 4; e += 32 * kWarps) {
        const int r = e / (HD / 4);
        float M = sR[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; w++) M = fmaxf(M, sR[w][r]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float ls = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = ex2(sR[w][r] - M);
            const float4 x = reinterpret_cast<const float4*>(so + w * 8 * HD)[e];
            v.x = fmaf(f, x.x, v.x);
            v.y = fmaf(f, x.y, v.y);
            v.z = fmaf(f, x.z, v.z);
            v.w = fmaf(f, x.w, v.w);
            ls = fmaf(f, sL[w][r], ls);
        }
        reinterpret_cast<float4*>(sc)[e] = v;
        if (e % (HD / 4) == 0) {
            sR[kWarps][r] = M;
            sL[kWarps][r] = ls;
        }
    }
    __syncthreads();
    if (cs > 1) {
        cluster_arrive();
        cluster_wait();
    }
    const uint32_t aR = smem_u32(&sR[kWarps][0]), aL = smem_u32(&sL[kWarps][0]), aO = smem_u32(sc);
    for (int e = (int)rank * 32 * kWarps + threadIdx.x; e < min(rows, 8) * (HD / 4); e += (int)cs * 32 * kWarps) {
        const int r = e / (HD / 4);
        float M = -FLT_MAX;
        for (uint32_t c = 0; c < cs; c++) M = fmaxf(M, ld_cluster(aR + 4 * r, c));
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float ls = 0.f;
        for (uint32_t c = 0; c < cs; c++) {
            const float f = ex2(ld_cluster(aR + 4 * r, c) - M);
            const float4 x = ld_cluster4(aO + 16 * e, c);
            v.x = fmaf(f, x.x, v.x);
            v.y = fmaf(f, x.y, v.y);
            v.z = fmaf(f, x.z, v.z);
            v.w = fmaf(f, x.w, v.w);
            ls = fmaf(f, ld_cluster(aL + 4 * r, c), ls);
        }
        const int rr = r0 + r;
        float* dst = a.out + ((int64_t)b * a.n_new + rr / mul) * a.out_stride + (int64_t)(kvh * mul + rr % mul) * HD +
                     4 * (e % (HD / 4));
        *reinterpret_cast<float4*>(dst) = make_float4(v.x / ls, v.y / ls, v.z / ls, v.w / ls);
    }
    if (cs > 1) {  // no CTA's shared memory goes while another reads it
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}

namespace {

using RowsFn = void (*)(AttendArgs);
RowsFn rows_fn(int hd) {
    switch (hd) {
        case 32: return kvq4_attend_rows_kernel<1>;
        case 64: return kvq4_attend_rows_kernel<2>;
        case 96: return kvq4_attend_rows_kernel<3>;
        case 128: return kvq4_attend_rows_kernel<4>;
        default: return kvq4_attend_rows_kernel<8>;
    }
}

size_t rows_smem(int nb) {
    const size_t ring = (size_t)kWarps * (kRing * tile_bytes(nb) + scale_bytes(nb)) + query_bytes(nb);
    const size_t merge = (size_t)(kWarps + 1) * 8 * 32 * nb * 4;
    return ring > merge ? ring : merge;
}

}  // namespace

int kvq4_attend(cn_ctx* ctx, const cn_kvq4& c, const float* q, int64_t q_stride, float* out, int64_t out_stride,
                const int* pos, const int* count, int batch, int n_new, int n_heads, float scale, const float2* rope,
                int neox, cudaStream_t st) {
    AttendArgs a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.pos = pos;
    a.count = count;
    a.rope = rope;
    a.kq = static_cast<const uint8_t*>(c.k_quants);
    a.vq = static_cast<const uint8_t*>(c.v_quants);
    a.kd = static_cast<const __half*>(c.k_scales);
    a.vd = static_cast<const __half*>(c.v_scales);
    a.seq_rows = kvq4_seq_rows(c);
    a.batch = batch;
    a.n_new = n_new;
    a.n_heads = n_heads;
    a.n_kv = c.n_kv_heads;
    a.ctx_len = c.ctx_len;
    a.neox = neox;
    a.mant = (float)frexp((double)scale * 1.4426950408889634, &a.exp);
    a.err = ctx->dev_err;
    const int64_t rows = (int64_t)n_new * (n_heads / c.n_kv_heads);
    const int64_t groups = (rows + 7) / 8, items = groups * c.n_kv_heads * batch;
    CN_CHECK(items < (1ll << 31) / kMaxCluster, CN_ERR_INVALID_ARG, "too many rows (%lld items)", (long long)items);
    const int nb = c.head_dim / 32;
    const int64_t room = (int64_t)ctx->sms * ctas_per_sm(nb);
    if (kvq4_prompt_ok(c.head_dim)) {
        // Which kernel: by both kernels' times over the cache's length, as the positions
        // are on the device; all figures are of full caches, and near the start of a long
        // one the other kernel may be the faster.  Here: 6 us for each round of CTAs and 23
        // positions of 128 values a ns.  One sequence, 64 heads over 8 of 128, 8 x tokens
        // rows, here / there: at 2000 positions 64 rows 16 / 20 us, 192 rows 27 / 24; at
        // 16000 64 rows 53 / 49, 96 rows 73 / 50, 192 rows 136 / 84.  Four sequences of 32
        // heads, 64 rows: at 100 29 / 16, at 2000 100 / 50, at 16000 540 / 287.
        int k, rc;
        double there = 0;
        if ((rc = kvq4_prompt_plan(ctx, rows, c.n_kv_heads, batch, c.head_dim, c.ctx_len, &k, &there))) return rc;
        const double here = 6e3 * (double)((items + room - 1) / room) + (double)items * c.ctx_len * c.head_dim / 2944.;
        if (there < here) return kvq4_attend_prompt(ctx, c.head_dim, k, a, st);
    }
    a.groups = (int)groups;
    // CTAs per item: the most that all run at once (8 x 64 heads of 128 at 131
    // thousand positions, 64 items: 372 us with 4, 301 with 6, 347 with 8), and
    // no more than give every warp a tile of the longest sequence
    const int64_t most = (c.ctx_len + kWarps * tile_pos(nb) - 1) / (kWarps * tile_pos(nb));
    int cluster = 1;
    for (int k : {2, 3, 4, 6, 8, kMaxCluster})
        if (k <= most && k * items <= room) cluster = k;
    RowsFn fn = rows_fn(c.head_dim);
    const size_t smem = rows_smem(nb);
    if (!(__atomic_load_n(&ctx->kvq4_ready, __ATOMIC_RELAXED) & (1u << nb))) {
        CN_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        CN_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        __atomic_fetch_or(&ctx->kvq4_ready, 1u << nb, __ATOMIC_RELAXED);
    }
    CN_CUDA(launch_cluster_k(false, cluster, fn, dim3((unsigned)(items * cluster)), dim3(32 * kWarps), smem, st, a));
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
    CN_CHECK((int64_t)n_new * (n_heads / cache->n_kv_heads) < (1ll << 31), CN_ERR_INVALID_ARG, "too many rows");
    CN_CHECK(q_stride >= qd && out_stride >= qd && q_stride % 4 == 0 && out_stride % 4 == 0, CN_ERR_INVALID_ARG,
             "q_stride %lld / out_stride %lld: at least %lld values and a multiple of 4", (long long)q_stride,
             (long long)out_stride, (long long)qd);
    CN_CHECK(((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_rope) % 16 == 0, CN_ERR_INVALID_ARG,
             "q, out and the rope table must be 16-byte aligned");
    CN_CHECK(isfinite(scale) && scale > 0.f, CN_ERR_INVALID_ARG, "scale must be finite and positive");
    CN_CHECK(rope_neox == 0 || rope_neox == 1, CN_ERR_INVALID_ARG, "rope_neox is 0 or 1");
    DeviceScope ds(ctx->device);
    return kvq4_attend(ctx, *cache, d_q, q_stride, d_out, out_stride, d_pos, d_count, batch, n_new, n_heads, scale,
                       reinterpret_cast<const float2*>(d_rope), rope_neox, (cudaStream_t)stream);
}
