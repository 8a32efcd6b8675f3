// Attention of drafted rows over a paged cache on the 5th-generation tensor cores: f16 / bf16 queries and pages,
// head_dim 64 or 128, pages of 8, 16, 32, 64 or a multiple of 128 slots.
//
// A CTA walks blocks of 128 keys for a tile of query rows (rows of the step x query heads of a group; what is missing is padding, which
// costs no memory traffic).  Two streams of four warps each have 128 rows, a score tile and an accumulator in tensor memory, so
// that one stream's exponentials run while the tensor cores work for the other.  Where sequences have few rows the streams share a tile of
// 128 and take its key blocks in turn; where they have more (TWO) each has a tile of its own and both use every block:
//
//   S_s = Q K_j^T          tcgen05.mma, operands in shared memory (TMA, 128-byte swizzle), f32 scores in tensor memory
//   P_s = 2^(S_s - m_s)    one thread per row; rounded to the pages' type, written over the scores in tensor memory
//   O_s += P_s V_j         tcgen05.mma, P from tensor memory, V from shared memory as it lies there (keys are the rows)
//
// and, where they shared the rows, the two accumulators are joined when the CTA leaves the unit.  A row's reference m_s follows its running maximum
// only when that has grown by more than 2^8 (weights then stay below 2^8 of the reference's and the accumulator is rarely rescaled: the
// result is the same quotient).  Sums, references and accumulators are f32; the weights are rounded once, to the type
// the tensor cores take.
//
// Warps: 0 TMA (every lane a box: a page's keys, 64 values of the head), 1 MMA issue, 2 the next segment's queries into the
// other query buffer, 3 the division of the work (Sched), 4-7 and 8-11 the streams.  Segments pass through a ring, so that loads and
// score products of the next one begin while the last one's results are stored.  Warps of a stream whose rows are all padding only keep step.
// Blocks that hold the rows' own tokens, or keys behind the last one, are masked, and their values in shared memory are cleaned
// first: rows behind the last key become zeros and values that are not finite are set aside (0 * inf would reach
// rows that do not see the token); the epilogue puts them in for the rows that do (put_odd).
//
// Every wait is bounded (about a second); on expiry a role leaves, waits (again with that limit) for the copies and products that it has in flight -
// they write the CTA's shared and tensor memory - and records DEV_TIMEOUT; all threads meet at the end and the tensor memory is freed.
#include "engine.h"
#include "tree_sched.cuh"

#include <cuda.h>

namespace ullm {
namespace {

constexpr int TM = 128, TK = 128, TT = 384;
// Places that a unit costs beside its blocks (64 sequences of one row: 2 for 125 us, 3 for 114, 4 for 112.6, 6 for 114); places that a CTA takes at least (one token: 2 for
// 12.3 us, 4 for 14.2, 6 for 16.1).
constexpr int T_COST = 4, T_MIN = 2;
constexpr int SEGS = 4;
template <int D> struct Cfg {
    static constexpr int ATOMS = D / 64;            // 64 values of a head: one 128-byte swizzle row
    static constexpr int TILE = ATOMS * TK * 128;   // bytes of 128 keys, and of 128 queries
    static constexpr int STAGES = D == 128 ? 5 : 10;
    static constexpr int SMEM = (2 + STAGES) * TILE + 1024;
    static constexpr uint32_t O_COL = 256;          // columns: scores 0 / 128, accumulators 256 / 256 + D
};

struct TcParams {
    TreeDev t;
    int *status;
    int box;       // keys of a TMA box
    int slot_dim;  // coordinate (1 or 2) of the slot; the other one is the head
    int q_box;     // rows of the step in a TMA box of queries; 0: queries through cp.async
    int team;      // logarithm of the CTAs of a team (Sched)
    int page_log;  // logarithm of the page size where it is below a block's keys
    int page_blocks; // blocks of a page where it is not
    long long wait;  // clock cycles after which a wait of the warps that enqueue loads and products gives up (the others: TREE_WAIT_CYCLES)
};
struct TcMaps {
    CUtensorMap k, v, q;
};

__device__ __forceinline__ bool mbar_test_wait(uint64_t *bar, uint32_t parity) { // (does not wait at all)
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// A converged warp waits; every lane gets the same answer, so that no lane leaves alone.  A limit of 0 only looks.
__device__ __forceinline__ bool wait_bounded(uint64_t *bar, uint32_t parity, long long limit = TREE_WAIT_CYCLES) {
    bool done = limit ? mbar_try_wait(bar, parity) : mbar_test_wait(bar, parity);
    const long long t0 = clock64();
    while (!__all_sync(0xffffffffu, done)) {
        if (!limit) return false;
#pragma unroll 1
        for (int i = 0; i < 64 && !done; ++i) done = mbar_try_wait(bar, parity);
        if (__any_sync(0xffffffffu, clock64() - t0 > limit)) return __all_sync(0xffffffffu, done);
    }
    return true;
}
// Waits for the last uses of a ring of barriers, `count` uses in all (uses i, i + stages, ... of barrier i).  Only where a role has given up.
__device__ __noinline__ void wait_for_last(uint64_t *bars, uint32_t count, uint32_t stages) {
    for (uint32_t i = count > stages ? count - stages : 0; i < count; ++i) wait_bounded(bars + i % stages, i / stages & 1);
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int c1, int c2, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(c1), "r"(c2), "r"(page), "r"(bar)
                 : "memory");
}
// 128-byte swizzle, version of sm_100.  Keys or rows as M / N with the head's values as K: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Values as N, keys as K: the next 64 values lie a whole atom further, the next 8 keys 1024 bytes further.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((TK * 128) >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D f32; A and B f16 (0) or bf16 (1); B transposed when its K is not the contiguous axis
template <typename T> constexpr uint32_t idesc(int n, bool b_mn) {
    constexpr uint32_t ty = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    return (1u << 4) | (ty << 7) | (ty << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
}
// Four MMAs (K = 16 each) by one elected lane of a converged warp, as one instruction sequence: issued one by one under a branch on the
// lane they took 100 cycles each.  A, B: descriptors that advance by `da`, `db` per step; `acc`: whether the first one adds to D.
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n.reg .pred pe, pf, pt;\n.reg .b64 a1, a2, a3, b1, b2, b3;\n"
                 "setp.ne.b32 pf, %4, 0;\nsetp.eq.b32 pt, 0, 0;\nelect.sync _|pe, 0xffffffff;\n"
                 "add.u64 a1, %1, 2;\nadd.u64 a2, %1, 4;\nadd.u64 a3, %1, 6;\nadd.u64 b1, %2, 2;\nadd.u64 b2, %2, 4;\nadd.u64 b3, %2, 6;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, pf;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, pt;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, pt;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, pt;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n.reg .pred pe, pf, pt;\n.reg .b32 a1, a2, a3;\n.reg .b64 b1, b2, b3;\n"
                 "setp.ne.b32 pf, %4, 0;\nsetp.eq.b32 pt, 0, 0;\nelect.sync _|pe, 0xffffffff;\n"
                 "add.u32 a1, %1, 8;\nadd.u32 a2, %1, 16;\nadd.u32 a3, %1, 24;\nadd.u64 b1, %2, 128;\nadd.u64 b2, %2, 256;\nadd.u64 b3, %2, 384;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, pf;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, pt;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, pt;\n"
                 "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, pt;\n}" ::"r"(d),
                 "r"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}
// Arrives on both barriers once the MMAs issued so far are complete.
__device__ __forceinline__ void commit2(uint64_t *x, uint64_t *y) {
    asm volatile("{\n.reg .pred pe;\nelect.sync _|pe, 0xffffffff;\n"
                 "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
                 "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}" ::"r"(smem_u32(x)),
                 "r"(smem_u32(y))
                 : "memory");
}
__device__ __forceinline__ void commit1(uint64_t *x) {
    asm volatile("{\n.reg .pred pe;\nelect.sync _|pe, 0xffffffff;\n"
                 "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(x))
                 : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Waits for a load of 32 values; their uses stay behind it.
__device__ __forceinline__ void wait_ld32(uint32_t *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
                   "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
                   "=r"(v[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                 "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]),
                 "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
                 "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { // two multiply-adds in one instruction
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b), "l"(*(unsigned long long *)&c));
    return *(float2 *)&r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b));
    return *(float2 *)&r;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Exponent bits all set in either half of a pair of 16-bit values: infinity or NaN
template <typename T> __device__ __forceinline__ uint32_t odd_halves(uint32_t w) { // 0xffff for each such half
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return ((w & E) == E ? 0xffffu : 0u) | ((w >> 16 & E) == E ? 0xffff0000u : 0u);
}
// f16 weights are held 2^6 larger, which keeps small ones out of the subnormals; at most 2^(6 + 8) < 65504.  bf16 values reach the end of the 32-bit range: weights
// 2^8 smaller are at most 1 however far the reference lags, so that a product is no larger than its value.
template <typename T> constexpr float lift() { return std::is_same<T, __half>::value ? 6.f : -8.f; }

// The part of a row's view that falls on keys key0 .. key0 + 31, as bits.
__device__ __forceinline__ uint32_t view_bits(const TreeDev &p, const SeqView &v, int i, int key0) {
    const int node0 = key0 - v.ctx, nodes = v.kv - v.ctx;
    uint32_t r;
    int limit; // nodes from node0 on that can be seen at all
    if (!p.mask) {
        r = 0xffffffffu, limit = min(i + 1, nodes) - node0;
    } else {
        const uint32_t *m = p.mask + (size_t)(v.r0 + i) * p.mask_words;
        const int w = node0 >> 5;
        const uint32_t lo = w < 0 ? 0xffffffffu : (w < p.mask_words ? m[w] : 0u), hi = w + 1 < 0 ? 0xffffffffu : (w + 1 < p.mask_words ? m[w + 1] : 0u);
        r = __funnelshift_r(lo, hi, node0 & 31), limit = nodes - node0;
    }
    return limit >= 32 ? r : (limit <= 0 ? 0u : r & ((1u << limit) - 1u));
}

// Place of the tile with the keys / values of block j of a segment of n blocks in the order in which tiles reach shared memory, which is
// that in which the tensor cores take them: K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1) where blocks alternate between the
// streams, K0 V0 K1 V1 ... where both streams take each.
template <bool TWO> __device__ __forceinline__ uint32_t k_tile(uint32_t j) { return TWO ? 2 * j : (j ? 2 * j - 1 : 0); }
template <bool TWO> __device__ __forceinline__ uint32_t v_tile(uint32_t j, uint32_t n) { return TWO ? 2 * j + 1 : (j + 1 == n ? 2 * n - 1 : 2 * j + 2); }

// Infinities and NaN among the values [c, c + 32) of tokens [first, last) that row `me` sees, in the place of the row's sums.  Rare, and out of the way.
template <typename T> __device__ __noinline__ void put_odd_at(const TreeDev &p, const SeqView &v, const T *q, int head, int me, int first, int last, int c, float *o) {
    const int *const table = p.blocks + (size_t)v.id * p.max_blocks;
    float sum[32];
    for (int e = 0; e < 32; ++e) sum[e] = 0.f;
    for (int token = first; token < last; ++token) {
        const int page = table[token / p.page_size];
        if ((unsigned)page >= (unsigned)p.n_pages || (token >= v.ctx && !sees(p, v, me, token - v.ctx))) continue;
        const long long at = page * p.page_stride + token % p.page_size * p.slot_stride + head * p.head_stride;
        const uint4 *const values = (const uint4 *)((const T *)p.v + at + c);
        uint32_t odd = 0;
        for (int i = 0; i < 4; ++i) {
            const uint4 x = values[i];
            odd |= odd_halves<T>(x.x) | odd_halves<T>(x.y) | odd_halves<T>(x.z) | odd_halves<T>(x.w);
        }
        if (!odd) continue;
        const bool none = has_no_weight(q, (const T *)p.k + at, p.dim, p.scale_log2);
        for (int e = 0; e < 32; ++e) {
            const float y = (float)((const T *)values)[e];
            if (!isfinite(y)) sum[e] += none ? NAN : y;
        }
    }
    for (int e = 0; e < 32; ++e)
        if (sum[e] != 0.f) o[e] = sum[e];
}
template <typename T>
__device__ __forceinline__ void put_odd(const TreeDev &p, const SeqView &v, const T *q, int head, int me, int first, int last, int c, float (&o)[32]) {
    float copy[32]; // (a register array cannot be indexed by the loops above)
#pragma unroll
    for (int e = 0; e < 32; ++e) copy[e] = o[e];
    put_odd_at<T>(p, v, q, head, me, first, last, c, copy);
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = copy[e];
}

template <typename T, int D, bool TWO> __global__ void __launch_bounds__(TT, 1) tree_attn_tc_kernel(const __grid_constant__ TcParams prm, const __grid_constant__ TcMaps maps) {
    using C = Cfg<D>;
    constexpr int NST = C::STAGES, ROWS = TWO ? 2 * TM : TM, STEP = TWO ? 1 : 2; // STEP: a stream takes every so many blocks
    extern __shared__ __align__(1024) uint8_t gsm[];
    uint8_t *const q_sm = (uint8_t *)(((uintptr_t)gsm + 1023) & ~(uintptr_t)1023), *const ring = q_sm + 2 * C::TILE;
    __shared__ uint64_t full[NST], empty[NST], s_full[2], p_full[2], o_done[2], h_full[2], q_full[2], q_empty[2], seg_full[SEGS], seg_empty[SEGS], x_full, epi_done, mma_done;
    __shared__ Seg segs[SEGS];
    __shared__ uint32_t tmem_s;
    const TreeDev &p = prm.t;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Set-up: warp 3 makes the barriers, tells the others and goes on to its part; they wait for it and the tensor memory.
    if (warp == 3) {
        if (lane == 0) {
            for (int i = 0; i < NST; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
            for (int s = 0; s < 2; ++s) {
                mbar_init(&s_full[s], 1), mbar_init(&h_full[s], 4), mbar_init(&p_full[s], 4), mbar_init(&o_done[s], 1);
                mbar_init(&q_full[s], 1), mbar_init(&q_empty[s], 8);
            }
            for (int i = 0; i < SEGS; ++i) mbar_init(&seg_full[i], 1), mbar_init(&seg_empty[i], 11);
            mbar_init(&x_full, 8), mbar_init(&epi_done, 8), mbar_init(&mma_done, 1);
            mbar_fence_init();
        }
        __syncwarp();
        asm volatile("barrier.cta.arrive 1, %0;" ::"n"(TT) : "memory");
    } else {
        if (warp == 0 && lane < 3) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &maps.k : (lane == 1 ? &maps.v : &maps.q)) : "memory");
        if (warp == 2) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        fence_before();
        asm volatile("barrier.cta.sync 1, %0;" ::"n"(TT) : "memory");
        fence_after();
    }
    pdl_wait_prior();
    pdl_launch_dependents();
    const uint32_t tmem = warp == 3 ? 0 : __shfl_sync(0xffffffffu, tmem_s, 0);
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) { return wait_bounded(bar, parity, prm.wait); };
    // the next segment of the ring; 0: no more
    uint32_t seg = 0;
    auto take = [&]() -> int {
        ok = wait_bounded(&seg_full[seg % SEGS], seg / SEGS & 1);
        return ok ? __shfl_sync(0xffffffffu, segs[seg % SEGS].count, 0) : 0;
    };
    auto give = [&]() { // this warp is done with the segment
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[seg % SEGS]);
        ++seg;
    };

    if (warp == 3) {
        // ---- division of the work ----
        if (lane == 0) p.meta[blockIdx.x * TREE_META] = make_int4(-1, 0, 0, 0);
        __syncwarp();
        Sched<ROWS, TK, T_COST, T_MIN> sched(p, prm.team);
        const bool some = sched.init();
        for (;; ++seg) {
            Seg next;
            next.count = 0;
            if (some) next = sched.next(p.meta + blockIdx.x * TREE_META);
            if (seg >= SEGS && !(ok = wait_bounded(&seg_empty[seg % SEGS], (seg / SEGS - 1) & 1))) break;
            if (lane == 0) {
                segs[seg % SEGS] = next;
                mbar_arrive(&seg_full[seg % SEGS]);
            }
            if (!next.count) break;
        }
    } else if (warp == 0) {
        // ---- TMA: lane -> (64 values, box of keys) ----
        const int atom = lane % C::ATOMS, part = lane / C::ATOMS, box = prm.box, parts = TK / box;
        const bool mine = part < parts;
        uint32_t tile0 = 0, asked = 0; // asked: tiles whose boxes are under way or there
        for (int n; (n = take()) != 0 && ok; give()) {
            const Seg &w = segs[seg % SEGS];
            const int key_end = w.key_end, h = w.h, first = w.blk * TK + part * box;
            // entries of the page table, 32 at a time and one such load ahead: a block has 1 to 16 of them
            const bool small = p.page_size < TK;
            auto entry_of = [&](int block) { return small ? block << (7 - prm.page_log) : (int)((unsigned)block / (unsigned)prm.page_blocks); }; // of a block's first key
            const int e0 = entry_of(w.blk), e_end = key_end <= 0 ? 0 : small ? (key_end + p.page_size - 1) >> prm.page_log : entry_of((key_end - 1) / TK) + 1;
            const int *const table = p.blocks + (size_t)w.id * p.max_blocks;
            auto entries = [&](int e) { return e + (int)lane < e_end ? table[e + lane] : 0; };
            int win = e0, now = entries(e0), ahead = entries(e0 + 32);
            auto page_of = [&](int j) { // page of this lane's box in block j of the segment
                const int first_e = entry_of(w.blk + j); // the same in every lane
                if (first_e >= win + 32) win += 32, now = ahead, ahead = entries(win + 32);
                return __shfl_sync(0xffffffffu, now, (first_e - win + (small ? part : 0)) & 31);
            };
            auto load = [&](const CUtensorMap *map, int j, uint32_t tile, int page) {
                const uint32_t st = tile % NST;
                if (tile >= NST && !wait(&empty[st], (tile / NST - 1) & 1)) return false;
                const int token = first + j * TK;
                const bool go = mine && token < key_end;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, go));
                if (lane == 0) mbar_arrive_expect_tx(&full[st], boxes * box * 128);
                __syncwarp();
                if (go) {
                    const int slot = prm.page_blocks <= 1 ? 0 : (int)((unsigned)(token / TK) % (unsigned)prm.page_blocks) * TK;
                    tma_box(smem_u32(ring) + st * C::TILE + atom * (TK * 128) + part * box * 128, map, atom * 64, prm.slot_dim == 1 ? slot : h,
                            prm.slot_dim == 1 ? h : slot, page, smem_u32(&full[st]));
                }
                asked = tile + 1;
                return true;
            };
            if (TWO) {
                for (int i = 0; i < n && ok; ++i) {
                    const int page = page_of(i);
                    ok = load(&maps.k, i, tile0 + k_tile<TWO>(i), page) && load(&maps.v, i, tile0 + v_tile<TWO>(i, n), page);
                }
            } else {
                int prev = 0;
                for (int i = 0; i <= n && ok; ++i) {
                    const int cur = i < n ? page_of(i) : 0;
                    if (i < n) ok = load(&maps.k, i, tile0 + k_tile<TWO>(i), cur);
                    if (i > 0 && ok) ok = load(&maps.v, i - 1, tile0 + v_tile<TWO>(i - 1, n), prev);
                    prev = cur;
                }
            }
            if (!ok) break;
            tile0 += 2 * n;
        }
        if (!ok) wait_for_last(full, asked, NST);
    } else if (warp == 2) {
        // ---- queries, as rows of the swizzled tile(s): a stream's 128 rows, or those that the streams share ----
        uint32_t asked = 0; // segments whose boxes are under way or there
        for (int n; (n = take()) != 0 && ok; give()) {
            const uint32_t b = TWO ? 0 : seg & 1, use = TWO ? seg : seg / 2; // TWO: both buffers in one go
            if (use && !(ok = wait_bounded(&q_empty[b], (use - 1) & 1))) break;
            const Seg &w = segs[seg % SEGS];
            const int rows = w.rows, group = p.group, token0 = w.r0 + w.row0 / group;
            if (prm.q_box) { // a box: q_box rows of the step x the group's heads x 64 values (rows behind the sequence's last are padding too)
                const int box_rows = prm.q_box * group, parts = (rows + box_rows - 1) / box_rows, boxes = parts * C::ATOMS;
                if (lane == 0) mbar_arrive_expect_tx(&q_full[b], boxes * box_rows * 128);
                __syncwarp();
                for (int i = lane; i < boxes; i += 32) {
                    const int atom = i % C::ATOMS, part = i / C::ATOMS, r = part * box_rows;
                    tma_box(smem_u32(q_sm) + (b + r / TM) * C::TILE + atom * (TM * 128) + r % TM * 128, &maps.q, atom * 64, 0, w.h, token0 + part * prm.q_box,
                            smem_u32(&q_full[b]));
                }
                asked = seg + 1;
            } else {
                constexpr int PIECES = D / 8, STRIDE = 32 / PIECES;
                const int piece = lane % PIECES, jump = STRIDE / group, left = STRIDE % group;
                int r = lane / PIECES, g = (w.row0 + r) % group;
                const T *src = (const T *)p.q + (w.r0 + (w.row0 + r) / group) * p.q_stride + ((long long)w.h * group + g) * D + piece * 8;
                const long long step = jump * p.q_stride + left * D, wrap = p.q_stride - (long long)group * D;
                const uint32_t dst = smem_u32(q_sm) + b * C::TILE + (piece / 8) * (TM * 128);
#pragma unroll 4
                for (; r < rows; r += STRIDE) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + r / TM * C::TILE + r % TM * 128 + (((piece % 8) ^ (r & 7)) << 4)), "l"(src) : "memory");
                    src += step, g += left;
                    if (g >= group) g -= group, src += wrap;
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[b]);
            }
        }
        if (!ok) wait_for_last(q_full, asked, TWO ? 1 : 2);
    } else if (warp == 1) {
        // ---- MMA issue: the whole warp with uniform control flow, one elected lane issues ----
        uint32_t tile0 = 0, done[2] = {0, 0};
        const uint32_t q0 = smem_u32(q_sm), r0 = smem_u32(ring);
        for (uint32_t n; (n = (uint32_t)take()) != 0 && ok; give()) {
            const uint64_t qd = desc_k_major(q0 + (TWO ? 0 : seg & 1) * C::TILE);
            if (!(ok = TWO ? wait(&q_full[0], seg & 1) : wait(&q_full[seg & 1], seg / 2 & 1))) break;
            // scores of block i for stream s; (the score tile's last user, P V of the stream's block before, was issued earlier and runs before)
            auto scores = [&](uint32_t s, uint32_t st) {
                const uint64_t kd = desc_k_major(r0 + st * C::TILE), q = qd + (TWO ? s : 0) * (C::TILE >> 4);
#pragma unroll
                for (int a = 0; a < C::ATOMS; ++a) mma4_ss(tmem + s * 128, q + a * (TM * 128 >> 4), kd + a * (TK * 128 >> 4), idesc<T>(TK, false), a > 0);
            };
            // P V.  Where both streams take every block the tensor cores set the pace and P comes in halves (262 -> 250 us for 12 x 64 drafted rows over
            // 4,000-16,000 tokens); where they alternate the second barrier costs more than it saves (64 decoded tokens: 125 -> 130 us).
            auto values = [&](uint32_t s, uint32_t st, bool add) {
                const uint64_t vd = desc_mn_major(r0 + st * C::TILE);
                if (!wait(TWO ? &h_full[s] : &p_full[s], done[s] & 1)) return false;
                fence_after();
                mma4_ts(tmem + C::O_COL + s * D, tmem + s * 128, vd, idesc<T>(D, true), add);
                if (TWO) {
                    if (!wait(&p_full[s], done[s] & 1)) return false;
                    fence_after();
                }
                ++done[s];
                mma4_ts(tmem + C::O_COL + s * D, tmem + s * 128 + 32, vd + 4 * 128, idesc<T>(D, true), 1);
                return true;
            };
            for (uint32_t i = 0; i <= n && ok; ++i) {
                const uint32_t kt = tile0 + k_tile<TWO>(i), ks = kt % NST, vt = tile0 + v_tile<TWO>(i - 1, n), vs = vt % NST; // (values of the block before)
                if (i == 1 && seg && !(ok = wait(&epi_done, (seg - 1) & 1))) break; // the accumulators have been read
                if (TWO) {
                    if (i > 0 && !(ok = wait(&full[vs], vt / NST & 1))) break;
#pragma unroll
                    for (uint32_t s = 0; s < 2; ++s) {
                        if (i > 0) {
                            if (!(ok = values(s, vs, i > 1))) break;
                            if (s == 1) commit2(&empty[vs], &o_done[s]);
                            else commit1(&o_done[s]);
                        }
                        if (i < n) {
                            if (s == 0 && !(ok = wait(&full[ks], kt / NST & 1))) break;
                            fence_after();
                            scores(s, ks);
                            if (s == 1) commit2(&empty[ks], &s_full[s]);
                            else commit1(&s_full[s]);
                        }
                    }
                } else {
                    if (i < n) {
                        if (!(ok = wait(&full[ks], kt / NST & 1))) break;
                        fence_after();
                        scores(i & 1, ks);
                        commit2(&empty[ks], &s_full[i & 1]);
                    }
                    if (i > 0) {
                        const uint32_t s = (i - 1) & 1;
                        if (!(ok = wait(&full[vs], vt / NST & 1) && values(s, vs, i > 2))) break;
                        commit2(&empty[vs], &o_done[s]);
                    }
                }
            }
            if (!ok) break;
            tile0 += 2 * n;
        }
        if (!ok) { // the products issued so far
            commit1(&mma_done);
            wait_for_last(&mma_done, 1, 1);
        }
    } else {
        // ---- the streams ----
        const uint32_t s = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t t_lane = tmem + (quarter * 32u << 16), t_s = t_lane + s * 128, t_o = t_lane + C::O_COL + s * D;
        uint32_t tile0 = 0, done[2] = {0, 0};
        const float scale = p.scale_log2;
        for (uint32_t n; (n = (uint32_t)take()) != 0 && ok; give()) {
            Seg &w = segs[seg % SEGS];
            SeqView v;
            v.r0 = w.r0, v.n = w.n, v.id = w.id, v.ctx = w.ctx, v.kv = w.kv;
            const int row0 = w.row0 + (TWO ? (int)s * TM : 0), rows = w.rows - (TWO ? (int)s * TM : 0), key_end = w.key_end, blk = w.blk; // this stream's
            const bool idle = (int)(quarter * 32) >= rows; // rows of padding: what they hold reaches no other row
            const int me = min((row0 + max(min((int)row, rows - 1), 0)) / p.group, v.n - 1); // this row's index in the sequence
            float m = -INFINITY, l = 0.f; // reference (a power of two), sum of weights
            for (uint32_t j = TWO ? 0 : s; j < n && ok; j += STEP) {
                const int key0 = (blk + j) * TK;
                const bool tail = key0 + TK > v.ctx;
                uint32_t bits[4];
                if (tail && !idle)
#pragma unroll
                    for (int c = 0; c < 4; ++c) bits[c] = view_bits(p, v, me, key0 + 32 * c);
                if (!(ok = wait_bounded(&s_full[s], done[s] & 1))) break;
                fence_after();
                if (!idle) {
                    if (tail) { // what a row does not see is masked where the scores lie
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t x[32];
                            const uint32_t see = c == 0 ? bits[0] : (c == 1 ? bits[1] : (c == 2 ? bits[2] : bits[3]));
                            tmem_ld32(t_s + 32 * c, x);
                            wait_ld32(x);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(see >> e & 1u)) x[e] = 0xff800000u;
                            tmem_st32(t_s + 32 * c, x);
                        }
                        wait_st();
                    }
                    // Two passes over the scores: the maximum, then the weights.  Reading tensor memory twice costs less than what 128 live values
                    // spill; the next 32 scores are on their way while 32 are worked on, and the tensor cores take the weights of
                    // the first 64 keys while those of the others are made.
                    float top[2] = {-INFINITY, -INFINITY};
                    uint32_t x[2][32];
                    tmem_ld32(t_s, x[0]);
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        wait_ld32(x[0]);
                        tmem_ld32(t_s + 64 * half + 32, x[1]);
#pragma unroll
                        for (int e = 0; e < 32; e += 2) top[e >> 1 & 1] = max3(top[e >> 1 & 1], __uint_as_float(x[0][e]), __uint_as_float(x[0][e + 1]));
                        wait_ld32(x[1]);
                        tmem_ld32(t_s + 64 - 64 * half, x[0]); // (the second time: the first ones again)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) top[e >> 1 & 1] = max3(top[e >> 1 & 1], __uint_as_float(x[1][e]), __uint_as_float(x[1][e + 1]));
                    }
                    const float block_max = fmaxf(top[0], top[1]) * scale - lift<T>();
                    if (__any_sync(0xffffffffu, block_max > m + 8.f)) {
                        const float to = block_max > m + 8.f ? block_max : m;
                        const float corr = m == to ? 1.f : ex2(m - to);
                        if (j >= STEP) {
                            if (!(ok = wait_bounded(&o_done[s], (done[s] - 1) & 1))) break; // P V of the stream's block before
                            fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                tmem_ld32(t_o + c, o);
                                wait_ld32(o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st32(t_o + c, o);
                            }
                        }
                        l *= corr, m = to;
                    }
                    const float sub = m == -INFINITY ? 0.f : m; // nothing seen yet: every weight is 2^-inf
                    const float2 scale2 = {scale, scale}, sub2 = {-sub, -sub};
                    float2 acc[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            wait_ld32(x[c]);
                            if (c == 0) tmem_ld32(t_s + 64 * half + 32, x[1]);
                            else if (half == 0) tmem_ld32(t_s + 64, x[0]);
                            uint32_t w16[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                float2 a = fma2(make_float2(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1])), scale2, sub2);
                                a.x = ex2(a.x), a.y = ex2(a.y);
                                acc[e & 1] = add2(acc[e & 1], a);
                                w16[e] = pack2<T>(a.x, a.y);
                            }
                            tmem_st16(t_s + 32 * half + 16 * c, w16); // over scores that have been read
                        }
                        if (TWO && half == 0 && !tail) {
                            wait_st();
                            fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&h_full[s]);
                        }
                    }
                    l += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
                    wait_st();
                }
                if (tail) { // clean the values of this block: thread = key
                    const uint32_t tile = tile0 + v_tile<TWO>(j, n), st = tile % NST, kr = tid & 127;
                    if (!(ok = wait_bounded(&full[st], tile / NST & 1))) break;
                    const int token = key0 + (int)kr;
                    if (token >= v.ctx) {
                        bool odd = false;
#pragma unroll 1
                        for (int a = 0; a < C::ATOMS; ++a)
#pragma unroll
                            for (int c = 0; c < 8; ++c) { // (the lanes of a row group on different banks)
                                uint4 *const at = (uint4 *)(ring + st * C::TILE + a * (TK * 128) + kr * 128 + ((c ^ (kr & 7)) << 4));
                                if (token >= key_end) {
                                    *at = make_uint4(0, 0, 0, 0);
                                } else {
                                    uint4 x = *at;
                                    const uint32_t o0 = odd_halves<T>(x.x), o1 = odd_halves<T>(x.y), o2 = odd_halves<T>(x.z), o3 = odd_halves<T>(x.w);
                                    if (o0 | o1 | o2 | o3) {
                                        x.x &= ~o0, x.y &= ~o1, x.z &= ~o2, x.w &= ~o3;
                                        *at = x;
                                        odd = true;
                                    }
                                }
                            }
                        if (odd) w.odd = 1;
                        fence_async();
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (TWO && (idle || tail)) mbar_arrive(&h_full[s]); // (a tail's values are clean only now)
                    mbar_arrive(&p_full[s]);
                }
                ++done[s];
            }
            if (!ok) break;
            // ---- join the streams' parts, store ----
            float2 a = make_float2(m, l), b = make_float2(-INFINITY, 0.f);
            if (TWO) {
                if (!(ok = wait_bounded(&o_done[s], (done[s] - 1) & 1))) break;
                fence_after();
            } else {
                done[1 - s] += s == 0 ? n / 2 : (n + 1) / 2;
                // all products of this segment that this stream waits for here were issued after the last use of the queries,
                // whose memory carries the references and sums from one stream to the other
                ok = wait_bounded(&o_done[0], (done[0] - 1) & 1) && (n < 2 || wait_bounded(&o_done[1], (done[1] - 1) & 1));
                if (!ok) break;
                float2 *const ml = (float2 *)(q_sm + (seg & 1) * C::TILE);
                ml[s * TM + row] = a;
                __syncwarp();
                if (lane == 0) mbar_arrive(&x_full);
                if (!(ok = wait_bounded(&x_full, seg & 1))) break;
                fence_after();
                a = ml[row];
                if (n >= 2) b = ml[TM + row];
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(&q_empty[TWO ? 0 : seg & 1]);
            if (!idle) {
                const float mm = fmaxf(a.x, b.x);
                const float wa = TWO ? 1.f : a.x == -INFINITY ? 0.f : ex2(a.x - mm), wb = b.x == -INFINITY ? 0.f : ex2(b.x - mm);
                const float ll = a.y * wa + b.y * wb;
                const bool whole = w.flags & 1, live = (int)row < rows, odd = w.odd;
                const int head = w.h;
                const int part_row = (TWO ? (int)s * TM : 0) + (int)row;
                float *const mine = part_of<ROWS>(p, blockIdx.x, w.flags >> 1);
                const float inv = ll == 0.f ? 0.f : 1.0f / ll;
                T *const out = (T *)p.out + (v.r0 + me) * p.out_stride + (head * p.group + (row0 + row) % p.group) * (long long)D;
                // the streams share a tile's columns, or each stores its own rows
#pragma unroll 1
                for (int c = TWO ? 0 : (int)s * (D / 2); c < (TWO ? D : (int)(s + 1) * (D / 2)); c += 32) {
                    uint32_t o0[32], o1[32];
                    __syncwarp(); // (rows part ways below)
                    tmem_ld32(TWO ? t_o + c : t_lane + C::O_COL + c, o0);
                    if (!TWO) tmem_ld32(t_lane + C::O_COL + D + c, o1);
                    wait_ld32(o0);
                    if (!TWO) wait_ld32(o1);
                    float o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = TWO ? __uint_as_float(o0[e]) : __uint_as_float(o0[e]) * wa + (n < 2 ? 0.f : __uint_as_float(o1[e]) * wb);
                    if (!live) continue;
                    float2 all[4]; // infinite or NaN where any of the values is (or where they pass the range together: then nothing is found below)
#pragma unroll
                    for (int e = 0; e < 4; ++e) all[e] = make_float2(o[2 * e], o[2 * e + 1]);
#pragma unroll
                    for (int e = 4; e < 16; ++e) all[e & 3] = add2(all[e & 3], make_float2(o[2 * e], o[2 * e + 1]));
                    all[0] = add2(add2(all[0], all[1]), add2(all[2], all[3]));
                    const bool bad = !(fabsf(all[0].x + all[0].y) < INFINITY) && ll == ll; // of tokens in front of the rows'; with a sum of weights that is NaN every value is
                    if (odd || bad)
                        put_odd<T>(p, v, (const T *)p.q + (v.r0 + me) * p.q_stride + (head * p.group + (row0 + row) % p.group) * (long long)D, head, me,
                                   bad ? blk * TK : max(v.ctx, blk * TK), min(key_end, (int)(blk + n) * TK), c, o);
                    if (whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint32_t y[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) y[k] = pack2<T>(ll == 0.f ? 0.f : o[e + 2 * k] * inv, ll == 0.f ? 0.f : o[e + 2 * k + 1] * inv);
                            *(uint4 *)(out + c + e) = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *(float4 *)(mine + (size_t)part_row * D + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                if (!whole && (TWO || s == 0) && live) *(float2 *)(mine + (size_t)ROWS * D + 2 * part_row) = make_float2(mm, ll);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&epi_done);
            tile0 += 2 * n;
        }
    }
    if (!ok) {
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); // (a stream may have left between a load and its use)
        wait_st();
        *(volatile int *)prm.status = DEV_TIMEOUT;
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
    static EncodeTiled fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess ? (EncodeTiled)f : nullptr;
    }();
    return fn;
}

// [values, slot and head (the nearer one first), page] of one layer; boxes of `box` slots x 64 values
bool encode_pool(const PoolDev &pool, int dtype, const uint8_t *base, int box, int *slot_dim, CUtensorMap *map) {
    const EncodeTiled enc = encoder();
    if (!enc) return false;
    const bool slot_first = pool.n_kv_head == 1 || (pool.page_size > 1 && pool.slot_stride < pool.head_stride);
    *slot_dim = slot_first ? 1 : 2;
    const cuuint64_t head_stride = (cuuint64_t)(pool.n_kv_head == 1 ? pool.page_stride : pool.head_stride) * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)pool.head_dim, (cuuint64_t)(slot_first ? pool.page_size : pool.n_kv_head),
                                (cuuint64_t)(slot_first ? pool.n_kv_head : pool.page_size), (cuuint64_t)pool.n_pages};
    const cuuint64_t strides[3] = {slot_first ? (cuuint64_t)pool.slot_stride * 2 : head_stride, slot_first ? head_stride : (cuuint64_t)pool.slot_stride * 2,
                                   (cuuint64_t)pool.page_stride * 2};
    const cuuint32_t boxes[4] = {64, slot_first ? (cuuint32_t)box : 1u, slot_first ? 1u : (cuuint32_t)box, 1}, one[4] = {1, 1, 1, 1};
    return enc(map, dtype == ULLM_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<uint8_t *>(base), dims, strides, boxes, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// [values, head of the group, group, row of the step]; boxes of q_box rows x all heads of a group x 64 values.  Such a box is a run of
// query rows in the tile's order when a tile holds whole rows of the step, and starts on a swizzle group.
bool encode_queries(const TreeDev &t, int dtype, int q_box, CUtensorMap *map) {
    const EncodeTiled enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)t.dim, (cuuint64_t)t.group, (cuuint64_t)t.n_kv, (cuuint64_t)t.n_rows};
    const cuuint64_t strides[3] = {(cuuint64_t)t.dim * 2, (cuuint64_t)t.group * t.dim * 2, (cuuint64_t)t.q_stride * 2};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)t.group, 1, (cuuint32_t)q_box}, one[4] = {1, 1, 1, 1};
    return t.q_stride < (1ll << 38) &&
           enc(map, dtype == ULLM_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<uint8_t *>(t.q), dims, strides, boxes, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool TWO> cudaError_t launch(const DeviceInfo &dev, const TcParams &prm, const TcMaps &maps, bool pdl, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(tree_attn_tc_kernel<T, D, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
    if (e != cudaSuccess) return e;
    if ((e = launch_kernel(tree_attn_tc_kernel<T, D, TWO>, dim3(dev.sm_count), dim3(TT), Cfg<D>::SMEM, st, pdl, prm, maps)) != cudaSuccess) return e;
    return launch_kernel(tree_join_kernel<T, TWO ? 2 * TM : TM>, dim3(dev.sm_count * JOIN_PER_SM<TWO ? 2 * TM : TM>), dim3(32 * JOIN_WARPS), 0, st, pdl, prm.t, dev.sm_count);
}
template <typename T> cudaError_t launch_any(const DeviceInfo &dev, int dim, bool two, const TcParams &prm, const TcMaps &maps, bool pdl, cudaStream_t st) {
    if (dim == 64) return two ? launch<T, 64, true>(dev, prm, maps, pdl, st) : launch<T, 64, false>(dev, prm, maps, pdl, st);
    return two ? launch<T, 128, true>(dev, prm, maps, pdl, st) : launch<T, 128, false>(dev, prm, maps, pdl, st);
}

} // namespace

bool tree_attn_tc_supported(const PoolDev &pool, int dtype) {
    if (dtype == ULLM_DTYPE_F32 || pool.elem_bytes != 2 || (pool.head_dim != 64 && pool.head_dim != 128)) return false;
    const int ps = pool.page_size; // a box of keys starts on a swizzle group of eight rows and lies in one page
    return ps % 128 == 0 || ps == 8 || ps == 16 || ps == 32 || ps == 64;
}
size_t tree_attn_tc_work(int sm_count, int dim) { return sizeof(float) * (size_t)sm_count * 2 * (2 * TM) * (dim + 2); }

cudaError_t launch_tree_attn_tc(const DeviceInfo &dev, const PoolDev &pool, int dtype, const TreeDev &t, int *d_status, long long wait_cycles, bool pdl, cudaStream_t st) {
    TcParams prm;
    TcMaps maps;
    prm.t = t, prm.status = d_status, prm.wait = wait_cycles, prm.box = pool.page_size < TK ? pool.page_size : TK, prm.slot_dim = 1;
    if (!encode_pool(pool, dtype, t.k, prm.box, &prm.slot_dim, &maps.k) || !encode_pool(pool, dtype, t.v, prm.box, &prm.slot_dim, &maps.v))
        return cudaErrorNotSupported;
    // Rows per sequence and key head on average (the lengths themselves are on the device; either way is right for any of them).
    const long long rows = ((long long)t.n_rows * t.group + t.n_seq - 1) / t.n_seq;
    // A tile of rows for each stream, or one for both: 390 rows on average 233 us against 239 to 266; 96 rows 27.1 against 23.9, 104 rows 136 against 104, 8 rows 160
    // against 113.
    const bool two = rows > TM;
    // CTAs of a team, where its members' tiles mostly exist: 390 rows 230 us with two, 248 without.
    prm.team = 0;
    while (two && prm.team < 2 && rows > (2 * TM << prm.team) * 5 / 4 && dev.sm_count >> (prm.team + 1) > 0) ++prm.team;
    prm.page_blocks = pool.page_size / TK, prm.page_log = 0;
    while (1 << prm.page_log < pool.page_size && prm.page_log < 7) ++prm.page_log;
    // query boxes of about a sequence's rows
    prm.q_box = 0;
    if (TM % t.group == 0) {
        int box = 1;
        while (box < t.n_rows / t.n_seq && box * t.group < TM) box *= 2;
        while (box * t.group % 8) box *= 2;
        if (encode_queries(t, dtype, box, &maps.q)) prm.q_box = box;
    }
    if (!prm.q_box) maps.q = maps.k; // (never used)
    return dtype == ULLM_DTYPE_F16 ? launch_any<__half>(dev, pool.head_dim, two, prm, maps, pdl, st) : launch_any<__nv_bfloat16>(dev, pool.head_dim, two, prm, maps, pdl, st);
}

} // namespace ullm
