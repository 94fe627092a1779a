// kvq4_prompt.cu -- attention over the 4-bit KV cache for many rows (prompts):
// the tcgen05 form of cn_kvq4_attend_dev.
//
// A CTA takes 128 rows (tokens x the query heads of one kv head) and walks the
// cache in tiles of 64 positions, K and V expanded from nibbles to fp16:
//   S = Q K^T:  Q [128 rows][hd] in tensor memory, K [64 positions][hd] in shared;
//   O = P V:    P [128 rows][64 positions] in tensor memory (in the scores' place),
//               V [hd][64 positions] in shared.
// Precision: q, k, v and the weights are pairs of fp16 halves (q and the weights to
// 22 bits; k and v, 15-bit products of a level and a scale, exactly), three MMAs each
// (lo hi + hi lo, then hi hi: the tensor cores truncate as they add, and lose less
// while the sum is small).  O is fresh for every tile and joined in fp32 registers for
// the same reason; that also leaves nothing to rescale in tensor memory.  A row's
// reference moves only when outgrown by 2^4.
//
// Bound: the tensor cores.  For a tile and hd = 128 they take 1590 cycles alone (48
// MMAs of 128 x 64 x 16 at 33) and 1880 next to the loads and stores of tensor memory;
// a tile takes 2030.  The rest must hide behind them, so each step has warps of its
// own (the instruction slots are 70 % full), four tiles are between their scores and
// their output, three expanded, and the output comes in halves, one read while the
// other is computed.  What it took, 64 query heads over 8 of hd 128, 1111 tokens at
// position 6000: 508 us at 1965 MHz, 470 TFLOP/s of the formula's 4 hd a pair, three
// times that as multiplied; call after call the power cap takes the clock to 1620 MHz,
// and it is 586 us, 407 TFLOP/s.  Other forms, at 1965 MHz: MMAs issued by a thread by
// itself, 84 cycles each: 831.  So with Q in shared memory and wide MMAs, fewer to issue:
// 641.  P in shared memory: 982.  Weights by eight warps on alternate tiles: 547.
// A CTA's first output comes 16600 cycles after its start, most of them the first
// pass through code that is in no instruction cache yet, and writing it takes 4000:
// 512 tokens at 0 (32 heads) take 24 us, of which their eight tiles are 9.
//
// Order of K's dimensions (any will do, if Q has the same) and V's rows (undone on
// the way out) follow the nibbles: K position kappa of a 64-wide half is
// (chunk g, word jj, nibble i, piece b & 1), V row n is (b & 1, i, g, jj), for value
// 32 b + 8 i + g, b = 2 jj + (b & 1).
#include <float.h>

#include "kvq4.cuh"
#include "kvq4_attend.cuh"

namespace cn {

namespace pr {

constexpr int kRows = 128, kPos = 64;
// warps 0-3 weights (a row a thread), 4-7 queries, then output, 8-11 K's expansion,
// 12-15 V's, 16 S, 17 loads, 18 O, 19 scales' ranges
constexpr int kThreads = 640;
constexpr int kRaw = 3;        // raw tiles in flight
constexpr int kBufs = 4;       // tiles between their scores and their output
constexpr int kStages = 3;     // expanded tiles
// Slots of words that pass between warps, more than any is ahead: a tile's weights
// are after the output of tile - kBufs, its scales' range after that of
// tile - kRaw - kStages - kBufs = tile - 10.
constexpr int kSlots = 8, kUndo = 16;
constexpr int kMaxCluster = 8;

template <int HD>
struct Geo {
    static constexpr int NB = HD / 32, W = NB / 2;  // blocks; 32-bit words per chunk
    static constexpr int kTile = kPos * HD * 2;     // bytes of one fp16 K or V tile
    static constexpr int kStage = 4 * kTile;        // K (hi, lo of each 64-wide part), V hi, V lo
    // rows of q, of the rope table and of the output in shared memory: 16 bytes
    // apart in the banks.  q's and the table's lie where the first V tile and what
    // follows it will; the output's (and a cluster's partials) where the first
    // stages were.
    static constexpr int kPitch = 4 * HD + 16, kQOff = 2 * kTile, kTabOff = kQOff + kRows * kPitch;
    static_assert(kTabOff + kRows * kPitch <= kStages * kStage, "queries");
    static constexpr int kRawTile = kPos * 36 * NB;
    static constexpr int kRawOff = kStages * kStage;
    static constexpr int kBarOff = kRawOff + kRaw * kRawTile;
    static constexpr int kRowOff = kBarOff + 768;  // per row: rescalings, the last reference and sum
    static constexpr int kSmem = kRowOff + kRows * (4 * kSlots + 8) + 1024;
    // tensor-memory columns: kBufs of S (the weights in its place, for 16 positions
    // 8 columns of halves and 8 of low halves); O; Q's halves, Q's low halves
    static constexpr int kS = 0, kO = kBufs * kPos, kQ = kO + HD;
    static constexpr int kCols = 512;
    static_assert(kQ + HD <= kCols, "tensor memory");
    static_assert(8 * (2 * kRaw + 4 * kStages + 3 * kBufs + 2 * kUndo + 6) + 8 + 8 * kUndo <= kRowOff - kBarOff, "barriers");
    static_assert(kBarOff % 8 == 0 && kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void ld32(uint32_t taddr, float* f) {
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void ld16(uint32_t taddr, float* f) {
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// D (+)= A (tensor memory) x B (shared memory)^T, kind::f16, fp32 accumulation
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// A K-major operand tile: rows of 128 bytes, 16-byte pieces at piece ^ (row & 7)
// (128-byte swizzle), 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// D fp32, A and B fp16, K-major, N columns, M = 128
__host__ __device__ constexpr uint32_t idesc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// Nibble i of both halves of x as level - 8, times d: hi + lo exactly.
__device__ __forceinline__ void expand(uint32_t x, int i, uint32_t d, uint32_t& hi, uint32_t& lo) {
    const uint32_t y = i >= 2 ? x >> 8 : x;
    const uint32_t v = (i & 1) ? odd_levels(y) : even_levels(y);
    hi = h2_mul(v, d);
    lo = h2_fms(v, d, hi);
}

}  // namespace pr

template <int HD>
__global__ void __launch_bounds__(pr::kThreads, 1) kvq4_attend_prompt_kernel(const AttendArgs a) {
    using namespace pr;
    using G = Geo<HD>;
    constexpr int NB = G::NB, W = G::W, RB = 16 * NB, SB = 2 * NB;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* raw_full = reinterpret_cast<uint64_t*>(smem + G::kBarOff);
    uint64_t* raw_empty = raw_full + kRaw;
    uint64_t* k_full = raw_empty + kRaw;
    uint64_t* v_full = k_full + kStages;
    uint64_t* k_empty = v_full + kStages;
    uint64_t* v_empty = k_empty + kStages;
    uint64_t* s_full = v_empty + kStages;
    uint64_t* p_full = s_full + kBufs;
    uint64_t* p_empty = p_full + kBufs;
    uint64_t* o_full = p_empty + kBufs;  // [2]
    uint64_t* o_empty = o_full + 2;      // [2]
    uint64_t* q_full = o_empty + 2;
    uint64_t* l_full = q_full + 1;
    uint64_t* u_full = l_full + 1;  // [2][kUndo]
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(u_full + 2 * kUndo);
    float* undo = reinterpret_cast<float*>(tmem_holder + 2);  // [2][kUndo] what K's and V's tiles were scaled down by
    float* slots = reinterpret_cast<float*>(smem + G::kRowOff);    // [kSlots][128] what a tile multiplies the row's output by
    float* mR = slots + kSlots * kRows;  // [128] the last references
    float* mL = mR + kRows;              // [128] sums of weights
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t cs = cluster_size(), rank = cluster_rank();

    // this cluster's 128 rows; the last tokens, which see most, first
    const int item = (int)(blockIdx.x / cs);
    const int bh = item % (a.batch * a.n_kv), grp = a.groups - 1 - item / (a.batch * a.n_kv);
    const int kvh = bh % a.n_kv, b = bh / a.n_kv;
    const int mul = a.n_heads / a.n_kv;
    int p0;
    const int n = kvq4_active(a.pos, a.count, b, a.n_new, a.ctx_len, p0);
    const int r0 = kRows * grp, rows = min(n * mul - r0, kRows);
    if (rows <= 0) return;  // (the whole cluster)
    const int len = p0 + (r0 + rows - 1) / mul + 1;  // positions any of the rows sees
    const int all = (len + kPos - 1) / kPos;
    const int tiles = all > (int)rank ? (all - (int)rank + (int)cs - 1) / (int)cs : 0;  // rank, rank + cs, ...
    const int64_t base = (int64_t)b * a.seq_rows + (int64_t)kvh * a.ctx_len;
    auto first_of = [&](int i) { return ((int)rank + i * (int)cs) * kPos; };

    if (warp == 0) {
        auto init = [&](uint64_t* bars, int n, int count) {
            if (lane < n) mbar_init(&bars[lane], count);
        };
        init(raw_full, kRaw, 1);
        init(raw_empty, kRaw, 9);
        init(k_full, 2 * kStages, 4);   // and v_full
        init(k_empty, 2 * kStages, 1);  // and v_empty
        init(s_full, kBufs, 1);
        init(p_full, kBufs, 4);
        init(p_empty, kBufs, 1);
        init(o_full, 2, 1);
        init(o_empty, 2, 4);
        init(q_full, 1, 4);
        init(l_full, 1, 4);
        init(u_full, 2 * kUndo, 1);
        fence_mbar_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                     "r"(G::kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // the rows' queries and their rows of the rope table, a row at a time: on their way
    const int tok0 = r0 / mul;
    if (warp >= 4 && warp < 8) {
        constexpr int kLanes = HD / 4;  // threads to a row
        const int k0 = (threadIdx.x & 127) / kLanes, e = threadIdx.x % kLanes;
        const float* q = a.q + (int64_t)b * a.n_new * a.q_stride + (int64_t)kvh * mul * HD + 4 * e;
        int tok = (r0 + k0) / mul, head = (r0 + k0) % mul;
        for (int k = k0; k < rows; k += kRows / kLanes) {
            copy16(smem + G::kQOff + k * G::kPitch + 16 * e, q + tok * a.q_stride + head * HD);
            for (head += kRows / kLanes; head >= mul; head -= mul) tok++;
        }
        if (a.rope)
            for (int k = k0; k <= (r0 + rows - 1) / mul - tok0; k += kRows / kLanes)
                copy16(smem + G::kTabOff + k * G::kPitch + 16 * e, a.rope + (int64_t)(p0 + tok0 + k) * (HD / 2) + 2 * e);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_holder;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !bar_wait(bar, parity & 1)) {
            ok = false;
            atomicOr(a.err, kErrTimeout);
        }
    };

    // Registers: 96 a thread at launch (480 for the five groups of four warps);
    // 112 + 184 + 64 + 80 + 32 = 472 once the last three have given theirs up.
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        if (warp == 17) {
            // ---- raw tiles ----
            if (lane == 0) {
                fence_proxy_async();
                int i = 0;
                for (; i < tiles; i++) {
                    const int s = i % kRaw;
                    if (i >= kRaw) wait(&raw_empty[s], (uint32_t)(i / kRaw - 1));
                    if (!ok) break;
                    const int first = first_of(i);
                    const int64_t row = base + first;
                    const int np = min(kPos, (len - first + 7) & ~7);  // (ctx_len is a multiple of 8)
                    uint8_t* d = smem + G::kRawOff + s * G::kRawTile;
                    mbar_expect_tx(&raw_full[s], (uint32_t)(np * 36 * NB));
                    bulk_load(d, a.kq + row * RB, np * RB, &raw_full[s]);
                    bulk_load(d + kPos * RB, a.vq + row * RB, np * RB, &raw_full[s]);
                    bulk_load(d + 2 * kPos * RB, a.kd + row * NB, np * SB, &raw_full[s]);
                    bulk_load(d + 2 * kPos * RB + kPos * SB, a.vd + row * NB, np * SB, &raw_full[s]);
                }
                // (whoever gave up, no copy outlives the CTA)
                for (int j = max(i - kRaw, 0); j < i; j++) bar_wait(&raw_full[j % kRaw], (uint32_t)(j / kRaw) & 1);
            }
        } else if (warp == 16 || warp == 18) {
            // ---- S, O.  The whole warp goes through the loops, with values that are
            // the same in all lanes, and one lane issues: 33 and 65 cycles an MMA of 64
            // and 128 columns, as the tensor cores take them; a thread by itself
            // issues one in 84 (50 with the loop unrolled). ----
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const int count = __shfl_sync(0xffffffffu, tiles, 0);
            const bool lead = elect_one();
            int i = 0;
            if (warp == 16) {
                constexpr uint32_t kN = idesc(kPos);
                if (count > 0) wait(q_full, 0);
                for (; i < count; i++) {
                    const int s = i % kStages, buf = i % kBufs;
                    wait(&k_full[s], (uint32_t)(i / kStages));
                    if (i >= kBufs) wait(&p_empty[buf], (uint32_t)(i / kBufs - 1));  // tile i - kBufs' weights lie there
                    if (!__all_sync(0xffffffffu, ok)) break;
                    fence_after();
                    const uint64_t kt = desc(smem_u32(smem + s * G::kStage));
                    const uint32_t d = tm + G::kS + buf * kPos;
                    // Qlo Khi, Qhi Klo, Qhi Khi
#pragma unroll
                    for (int m = 0; m < 3; m++)
#pragma unroll
                        for (int kk = 0; kk < HD / 16; kk++)
                            if (lead)
                                mma_ts(d, tm + G::kQ + (m == 0 ? HD / 2 : 0) + 8 * kk,
                                       kt + (m == 1 ? kPos * 128 / 16 : 0) + (kk >> 2) * (2 * kPos * 128 / 16) + 2 * (kk & 3),
                                       kN, m + kk != 0);
                    if (lead) {
                        commit(&s_full[buf]);
                        commit(&k_empty[s]);
                    }
                    __syncwarp();
                }
                // (whoever gave up, no MMA outlives its tensor memory)
                if (i > 0) bar_wait(&s_full[(i - 1) % kBufs], (uint32_t)((i - 1) / kBufs) & 1);
            } else {
                constexpr uint32_t kN = idesc(HD / 2);
                for (; i < count; i++) {
                    const int s = i % kStages, buf = i % kBufs;
                    wait(&v_full[s], (uint32_t)(i / kStages));
                    wait(&p_full[buf], (uint32_t)(i / kBufs));
                    // the output in halves: one is read while the other is computed
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (i > 0) wait(&o_empty[h], (uint32_t)(i - 1));
                        if (!__all_sync(0xffffffffu, ok)) break;
                        fence_after();
                        const uint64_t vt = desc(smem_u32(smem + s * G::kStage + 2 * G::kTile)) + h * (HD / 2 * 128 / 16);
                        const uint32_t d = tm + G::kO + h * (HD / 2), p = tm + G::kS + buf * kPos;
#pragma unroll
                        for (int m = 0; m < 3; m++)
#pragma unroll
                            for (int kk = 0; kk < kPos / 16; kk++)
                                if (lead)
                                    mma_ts(d, p + 16 * kk + (m == 0 ? 8 : 0), vt + (m == 1 ? G::kTile / 16 : 0) + 2 * kk, kN,
                                           m + kk != 0);
                        if (lead) commit(&o_full[h]);
                    }
                    if (!__all_sync(0xffffffffu, ok)) break;
                    if (lead) {
                        commit(&v_empty[s]);
                        commit(&p_empty[buf]);
                    }
                    __syncwarp();
                }
                if (i > 0) bar_wait(&o_full[1], (uint32_t)(i - 1) & 1);
                if (i < count) bar_wait(&o_full[0], (uint32_t)i & 1);
            }
        } else {
            // ---- what a tile's scales are multiplied by: those from 2^12 on would take fp16
            // products past its range, and a tile of K or V that has one counts 2^-4 times ----
            for (int i = 0, rs = 0, ph = 0; i < tiles; i++) {
                wait(&raw_full[rs], ph);
                const uint4* sc = reinterpret_cast<const uint4*>(smem + G::kRawOff + rs * G::kRawTile + 2 * kPos * RB);
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    uint32_t mx = 0;
#pragma unroll
                    for (int e = lane; e < kPos * NB / 8; e += 32) {  // eight scales
                        const uint4 v = sc[kv * (kPos * NB / 8) + e];
                        const int n = min(8, (len - first_of(i)) * NB - 8 * e);  // (rows past the end hold anything)
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int k = 0; k < 4; k++) mx = __vmaxu2(mx, 2 * k < n ? w[k] & 0x7FFF7FFFu : 0u);
                    }
                    const bool big = __any_sync(0xffffffffu, max(mx & 0xFFFFu, mx >> 16) >= 0x6C00u);
                    if (lane == 0) {
                        undo[kUndo * kv + i % kUndo] = big ? 16.f : 1.f;
                        mbar_arrive(&u_full[kUndo * kv + i % kUndo]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_empty[rs]);
                if (++rs == kRaw) rs = 0, ph ^= 1;
            }
        }
    } else if (warp >= 8) {
        // ---- expansion: K by warps 8-11, V by 12-15 ----
        const int tid = threadIdx.x & 127;
        const int kv = warp >= 12;
        auto shrink_of = [&](int i) {  // (rows and their scales have landed)
            wait(&u_full[kUndo * kv + i % kUndo], (uint32_t)(i / kUndo));
            return undo[kUndo * kv + i % kUndo] == 1.f ? 0x3C003C00u : 0x2C002C00u;
        };
        // the next tile's places in the rings, and the parities of their barriers
        auto step = [&](int& rs, int& ph, int& s, int& sp) {
            if (++rs == kRaw) rs = 0, ph ^= 1;
            if (++s == kStages) s = 0, sp ^= 1;
        };
        if (!kv) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
            // position p, chunks 4 hf .. + 3 (each W 16-byte pieces)
            const int p = tid & 63, hf = tid >> 6;
            for (int i = 0, rs = 0, ph = 0, s = 0, sp = 1; i < tiles; i++) {
                const uint8_t* raw = smem + G::kRawOff + rs * G::kRawTile;
                wait(&raw_full[rs], ph);
                const uint32_t shrink = shrink_of(i);
                const bool in = first_of(i) + p < len;
                const uint32_t* sc = reinterpret_cast<const uint32_t*>(raw + 2 * kPos * RB + p * SB);
                uint32_t d[W];
#pragma unroll
                for (int j = 0; j < W; j++) d[j] = in ? h2_mul(sc[j], shrink) : 0u;
                if (i == 1) wait(q_full, 0);  // (the queries lay there)
                if (i >= kStages) wait(&k_empty[s], sp);
#pragma unroll 1
                for (int j = 0; j < W; j++) {
                    const uint4 u = reinterpret_cast<const uint4*>(raw + p * RB + hf * (RB / 2))[j];
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
                    const int first16 = hf * 4 * W + 4 * j;  // the row's 16-byte pieces from here on (8 to a 64-wide part)
                    uint8_t* stage = smem + s * G::kStage + (first16 >> 3) * (2 * kPos * 128) + p * 128;
                    const int x = ((first16 & 7) ^ (p & 7)) << 4;
#pragma unroll
                    for (int c = 0; c < 4; c++) {  // word c % W of chunk (4 j + c) / W of this half
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) expand(w[c], e, d[c % W], hi[e], lo[e]);
                        uint8_t* t = stage + (x ^ (c << 4));
                        *reinterpret_cast<uint4*>(t) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4*>(t + kPos * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&k_full[s]);
                    mbar_arrive(&raw_empty[rs]);
                }
                step(rs, ph, s, sp);
            }
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
            // eight positions 8 k .. + 7, word gw = (g, jj); with one word a chunk,
            // nibbles in two halves
            const int gw = tid & (8 * W - 1), k = (tid / (8 * W)) & 7;
            constexpr int NI = 2 * W;  // nibbles a thread takes
            const int i0 = W == 2 ? 0 : (tid >> 6) * 2;
            for (int i = 0, rs = 0, ph = 0, s = 0, sp = 1; i < tiles; i++) {
                const int first = first_of(i) + 8 * k;
                const uint8_t* raw = smem + G::kRawOff + rs * G::kRawTile;
                wait(&raw_full[rs], ph);
                const uint32_t shrink = shrink_of(i);
                const uint8_t* q = raw + kPos * RB + 8 * k * RB + 4 * gw;
                const uint8_t* sc = raw + 2 * kPos * RB + kPos * SB + 8 * k * SB + 4 * (gw % W);
                uint32_t w[8], d[8];
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    w[u] = *reinterpret_cast<const uint32_t*>(q + u * RB);
                    d[u] = *reinterpret_cast<const uint32_t*>(sc + u * SB);
                    d[u] = first + u < len ? h2_mul(d[u], shrink) : 0u;  // (rows past the end hold anything)
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_empty[rs]);
                if (i == 0) wait(q_full, 0);
                if (i >= kStages) wait(&v_empty[s], sp);
                uint8_t* stage = smem + s * G::kStage + 2 * G::kTile;
#pragma unroll 1
                for (int pb = 0; pb < 2; pb++)
#pragma unroll
                    for (int e = 0; e < NI; e++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            uint32_t x = __byte_perm(w[2 * u], w[2 * u + 1], pb ? 0x7632u : 0x5410u);
                            const uint32_t dd = __byte_perm(d[2 * u], d[2 * u + 1], pb ? 0x7632u : 0x5410u);
                            if (W == 1 && i0) x >>= 8;  // nibbles 2, 3
                            expand(x, e, dd, hi[u], lo[u]);
                        }
                        const int row = (pb * 4 + i0 + e) * (8 * W) + gw;
                        uint8_t* t = stage + row * 128 + ((k ^ (row & 7)) << 4);
                        *reinterpret_cast<uint4*>(t) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4*>(t + G::kTile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[s]);
                step(rs, ph, s, sp);
            }
        }
    } else {
        const int r = threadIdx.x & (kRows - 1);  // this thread's row
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const int rr = r0 + min(r, rows - 1), tok = rr / mul;
        if (warp >= 4) {
            // ---- output ----
            asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
            float o[HD];
            {
                // first the row's query: rotated, scaled to [2^13, 2^15], in K's order
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const uint8_t* x = smem + G::kQOff + min(r, rows - 1) * G::kPitch;
#pragma unroll
                for (int e = 0; e < HD / 4; e++) {
                    const float4 v = reinterpret_cast<const float4*>(x)[e];
                    o[4 * e] = v.x, o[4 * e + 1] = v.y, o[4 * e + 2] = v.z, o[4 * e + 3] = v.w;
                }
                if (a.rope) {
                    const float4* tab = reinterpret_cast<const float4*>(smem + G::kTabOff + (tok - tok0) * G::kPitch);
                    auto turn = [](float& u, float& v, float c, float s) {
                        const float t = __fsub_rn(__fmul_rn(u, c), __fmul_rn(v, s));
                        v = __fadd_rn(__fmul_rn(u, s), __fmul_rn(v, c));
                        u = t;
                    };
                    if (a.neox) {
#pragma unroll
                        for (int e = 0; e < HD / 2; e += 2) {
                            const float4 t = tab[e / 2];
                            turn(o[e], o[e + HD / 2], t.x, t.y);
                            turn(o[e + 1], o[e + 1 + HD / 2], t.z, t.w);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < HD / 2; e += 2) {
                            const float4 t = tab[e / 2];
                            turn(o[2 * e], o[2 * e + 1], t.x, t.y);
                            turn(o[2 * e + 2], o[2 * e + 3], t.z, t.w);
                        }
                    }
                }
                float amax = 0.f, sc, inv;
#pragma unroll
                for (int e = 0; e < HD; e++) amax = fmaxf(amax, fabsf(o[e]));
                row_pow2_scale(amax, sc, inv);
                mR[r] = score_factor(inv, a.exp);  // for the weights' warps
                sc *= a.mant;
#pragma unroll
                for (int c = 0; c < HD / 32; c++) {  // 32 dimensions: four pieces of 8
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int g = (4 * c + k) / W, jj = (4 * c + k) % W;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int e = 64 * jj + 8 * i + g;  // and the next block's
                            split2(o[e] * sc, o[e + 32] * sc, hi[4 * k + i], lo[4 * k + i]);
                        }
                    }
                    st16(tmem + lane_off + G::kQ + 16 * c, hi);
                    st16(tmem + lane_off + G::kQ + HD / 2 + 16 * c, lo);
                }
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
#pragma unroll
            for (int e = 0; e < HD; e++) o[e] = 0.f;
            for (int i = 0; i < tiles; i++) {
                float up = 1.f, vm = 1.f;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    wait(&o_full[h], (uint32_t)i);
                    fence_after();
                    if (h == 0) {  // (the tile's words are there: the product came after them)
                        up = slots[(i % kSlots) * kRows + r];
                        vm = undo[kUndo + i % kUndo];
                    }
                    float t[2][16];
                    const uint32_t col = tmem + lane_off + G::kO + h * (HD / 2);
                    ld16(col, t[0]);
                    if (!__all_sync(0xffffffffu, up == 1.f)) {
#pragma unroll
                        for (int e = 0; e < HD / 2; e++) o[h * (HD / 2) + e] *= up;
                    }
#pragma unroll
                    for (int c = 0; c < HD / 32; c++) {
                        wait_ld();
                        if (c + 1 < HD / 32) ld16(col + 16 * (c + 1), t[(c + 1) & 1]);
                        else {
                            fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&o_empty[h]);
                        }
                        const float* x = t[c & 1];
                        float* y = o + h * (HD / 2) + 16 * c;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 v = fma2(make_float2(x[e], x[e + 1]), make_float2(vm, vm), make_float2(y[e], y[e + 1]));
                            y[e] = v.x, y[e + 1] = v.y;
                        }
                    }
                }
            }
            wait(l_full, 0);
            const float inv = cs > 1 ? 1.f : 1.f / mL[r];
            uint8_t* row = smem + r * G::kPitch;
#pragma unroll
            for (int m = 0; m < HD / 4; m++) {
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int e = 4 * m + u, bl = e / 32, i = (e / 8) % 4, g = e % 8;
                    v[u] = o[((bl & 1) * 4 + i) * (8 * W) + g * W + (bl >> 1)] * inv;
                }
                *reinterpret_cast<float4*>(row + 16 * m) = make_float4(v[0], v[1], v[2], v[3]);
            }
            if (cs == 1) {  // a row at a time
                constexpr int kLanes = HD / 4;
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const int k0 = r / kLanes, e = r % kLanes;
                float* dst = a.out + (int64_t)b * a.n_new * a.out_stride + (int64_t)kvh * mul * HD + 4 * e;
                int t = (r0 + k0) / mul, head = (r0 + k0) % mul;
                for (int k = k0; k < rows; k += kRows / kLanes) {
                    *reinterpret_cast<float4*>(dst + t * a.out_stride + head * HD) =
                        *reinterpret_cast<const float4*>(smem + k * G::kPitch + 16 * e);
                    for (head += kRows / kLanes; head >= mul; head -= mul) t++;
                }
            }
        } else {
            // ---- weights ----
            asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
            float R = -FLT_MAX, l = 0.f;
            const int limit = p0 + tok;
            wait(q_full, 0);
            const float factor = mR[r];
            const int seen_by_all = p0 + r0 / mul + 1;
            float x[64];  // a tile's scores, on their way while the last tile's weights are stored
            auto fetch = [&](int i) {
                wait(&s_full[i % kBufs], (uint32_t)(i / kBufs));
                fence_after();
                const uint32_t sc = tmem + lane_off + G::kS + (i % kBufs) * kPos;
                ld32(sc, x);
                ld32(sc + 32, x + 32);
            };
            if (tiles > 0) fetch(0);
            for (int i = 0; i < tiles; i++) {
                const int buf = i % kBufs, first = first_of(i);
                const uint32_t sc = tmem + lane_off + G::kS + buf * kPos;
                const float f = factor * undo[i % kUndo];  // (there since before K was expanded)
                const bool hide = first + kPos > seen_by_all;
                float top = -INFINITY, top2 = -INFINITY, move = 1.f;
                wait_ld();
                if (hide) {
#pragma unroll
                    for (int e = 0; e < 64; e++)
                        if (first + e > limit) x[e] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 32; e++) top = fmaxf(top, x[e]), top2 = fmaxf(top2, x[32 + e]);
                top = fmaxf(top, top2);
                if (top * f - R > kPeak + kLazy) {
                    const float to = reference(top * f);
                    move = ex2(R - to);
                    R = to;
                }
                // 16 scores at a time: weights, and their halves in the scores' place
                float2 part = make_float2(0.f, 0.f);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float2 v = fma2(make_float2(x[16 * c + e], x[16 * c + e + 1]), make_float2(f, f), make_float2(-R, -R));
                        v = make_float2(ex2(v.x), ex2(v.y));
                        part = add2(part, v);
                        split2(v.x, v.y, w[e / 2], w[8 + e / 2]);
                    }
                    st16(sc + 16 * c, w);
                }
                const float sum = part.x + part.y;
                l = l * move + sum;
                slots[(i % kSlots) * kRows + r] = move;
                if (i + 1 < tiles) fetch(i + 1);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[buf]);
            }
            mR[r] = R;
            mL[r] = l;
            __syncwarp();
            if (lane == 0) mbar_arrive(l_full);
        }
    }
    // every MMA is done and every copy landed
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 16)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::kCols) : "memory");
    if (cs > 1) {
        // the partials meet, each CTA adding up a share
        cluster_arrive();
        cluster_wait();
        const uint32_t aO = smem_u32(smem), aR = smem_u32(mR), aL = smem_u32(mL);
        for (int e = (int)rank * kThreads + threadIdx.x; e < rows * (HD / 4); e += (int)cs * kThreads) {
            const int r = e / (HD / 4), at = r * G::kPitch + 16 * (e % (HD / 4)), rr = r0 + r;
            float M = -FLT_MAX, ls = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t c = 0; c < cs; c++) M = fmaxf(M, ld_cluster(aR + 4 * r, c));
            for (uint32_t c = 0; c < cs; c++) {
                const float f = ex2(ld_cluster(aR + 4 * r, c) - M);
                const float4 x = ld_cluster4(aO + at, c);
                v.x = fmaf(f, x.x, v.x);
                v.y = fmaf(f, x.y, v.y);
                v.z = fmaf(f, x.z, v.z);
                v.w = fmaf(f, x.w, v.w);
                ls = fmaf(f, ld_cluster(aL + 4 * r, c), ls);
            }
            float* dst = a.out + ((int64_t)b * a.n_new + rr / mul) * a.out_stride + (int64_t)(kvh * mul + rr % mul) * HD;
            reinterpret_cast<float4*>(dst)[e % (HD / 4)] = make_float4(v.x / ls, v.y / ls, v.z / ls, v.w / ls);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}

bool kvq4_prompt_ok(int hd) { return hd == 64 || hd == 128; }

using PromptFn = void (*)(AttendArgs);
static PromptFn prompt_fn(int hd) { return hd == 64 ? kvq4_attend_prompt_kernel<64> : kvq4_attend_prompt_kernel<128>; }
static int prompt_smem(int hd) { return hd == 64 ? pr::Geo<64>::kSmem : pr::Geo<128>::kSmem; }
static int64_t prompt_items(int64_t rows, int n_kv, int batch) {
    return (rows + pr::kRows - 1) / pr::kRows * n_kv * batch;
}

// The time in ns that a call takes over the cache's length, and the CTAs per item for
// which it is shortest (four tiles for each at least): per round of clusters 12 us, 5
// more above one CTA, and 1.08 us a tile of 64 x 128 values.  64 query heads over 8:
// 16 tokens at 30000 80 us with 8 CTAs, 170 by the kernel for few rows; 296 at 6000
// (152 items on 148 SMs) 195 us with 2, 227 with one.
int kvq4_prompt_plan(cn_ctx* ctx, int64_t rows, int n_kv, int batch, int hd, int ctx_len, int* cluster, double* time) {
    int* fit = ctx->kvq4_fit[hd == 128];
    const uint32_t bit = 1u << (hd == 64 ? 24 : 25);
    if (!(__atomic_load_n(&ctx->kvq4_ready, __ATOMIC_ACQUIRE) & bit)) {
        const PromptFn fn = prompt_fn(hd);
        CN_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, prompt_smem(hd)));
        for (int i = 0; i < 4; i++) {
            cudaLaunchAttribute at = {};
            at.id = cudaLaunchAttributeClusterDimension;
            at.val.clusterDim.x = 1u << i;
            at.val.clusterDim.y = at.val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)(ctx->sms + 7) / 8 * 8);
            cfg.blockDim = dim3(pr::kThreads);
            cfg.dynamicSmemBytes = (size_t)prompt_smem(hd);
            cfg.attrs = &at;
            cfg.numAttrs = 1;
            int n = 0;
            CN_CUDA(cudaOccupancyMaxActiveClusters(&n, fn, &cfg));
            __atomic_store_n(&fit[i], n, __ATOMIC_RELAXED);
        }
        __atomic_fetch_or(&ctx->kvq4_ready, bit, __ATOMIC_RELEASE);
    }
    const int64_t items = prompt_items(rows, n_kv, batch), tiles = (ctx_len + pr::kPos - 1) / pr::kPos;
    *cluster = 0;
    for (int i = 0, k = 1; k <= pr::kMaxCluster && (k == 1 || 4 * k <= tiles); i++, k *= 2) {
        const int n = __atomic_load_n(&fit[i], __ATOMIC_RELAXED);
        if (k > 1 && n < 1) continue;
        const double t = (double)((items + n - 1) / (n > 0 ? n : 1)) *
                         ((k > 1 ? 17e3 : 12e3) + (double)((tiles + k - 1) / k) * 8.4 * hd);
        if (*cluster == 0 || t < *time) {
            *time = t;
            *cluster = k;
        }
    }
    return CN_OK;
}

int kvq4_attend_prompt(cn_ctx* ctx, int hd, int cluster, AttendArgs a, cudaStream_t st) {
    using namespace pr;
    const int64_t rows = (int64_t)a.n_new * (a.n_heads / a.n_kv), items = prompt_items(rows, a.n_kv, a.batch);
    CN_CHECK(items < (1ll << 31) / kMaxCluster, CN_ERR_INVALID_ARG, "too many rows (%lld items)", (long long)items);
    a.groups = (int)((rows + kRows - 1) / kRows);
    CN_CUDA(launch_cluster_k(false, cluster, prompt_fn(hd), dim3((unsigned)(items * cluster)), dim3(kThreads),
                             (size_t)prompt_smem(hd), st, a));
    return CN_OK;
}

}  // namespace cn
