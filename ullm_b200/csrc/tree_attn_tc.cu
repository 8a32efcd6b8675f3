// Attention of drafted rows over a paged cache on the 5th-generation tensor cores: f16 / bf16 queries and pages,
// head_dim 64 or 128, pages of 8, 16, 32, 64 or a multiple of 128 slots.
//
// A CTA takes 128 query rows (rows of the step x query heads of a group; what is missing is padding, which costs no
// memory traffic) and walks blocks of 128 keys.  Two streams of four warps take the blocks in turn, each with a score
// tile and an accumulator of its own in tensor memory, so that one stream's exponentials run while the tensor cores work for the other:
//
//   S_s = Q K_j^T          tcgen05.mma, operands in shared memory (TMA, 128-byte swizzle), f32 scores in tensor memory
//   P_s = 2^(S_s - m_s)    one thread per row; rounded to the pages' type, written over the scores in tensor memory
//   O_s += P_s V_j         tcgen05.mma, P from tensor memory, V from shared memory as it lies there (keys are the rows)
//
// and the two accumulators are joined when the CTA leaves the unit.  A row's reference m_s follows its running maximum
// only when that has grown by more than 2^8 (weights then stay below 2^8 and the accumulator is rarely rescaled: the
// result is the same quotient).  Sums, references and accumulators are f32; the weights are rounded once, to the type
// the tensor cores take.
//
// Warps: 0 TMA (every lane a box: a page's keys, 64 values of the head), 1 MMA issue, 2 tensor memory, 4-7 and 8-11 the streams.
// Blocks that hold the rows' own tokens, or keys behind the last one, are masked, and their values in shared memory are cleaned
// first: rows behind the last key become zeros and values that are not finite are set aside (0 * inf would reach
// rows that do not see the token); the epilogue adds them for the rows that do.
//
// Every wait is bounded (about a second); on expiry a role records DEV_TIMEOUT and leaves, all threads meet at the end and
// the tensor memory is freed.
#include "engine.h"
#include "tree_sched.cuh"

#include <cuda.h>

namespace ullm {
namespace {

constexpr int TM = 128, TK = 128, TT = 384;
template <int D> struct Cfg {
    static constexpr int ATOMS = D / 64;            // 64 values of a head: one 128-byte swizzle row
    static constexpr int TILE = ATOMS * TK * 128;   // bytes of 128 keys
    static constexpr int STAGES = D == 128 ? 6 : 10;
    static constexpr int SMEM = ATOMS * TM * 128 + STAGES * TILE + 1024;
    static constexpr uint32_t O_COL = 256;          // columns: scores 0 / 128, accumulators 256 / 256 + D
};

struct TcParams {
    TreeDev t;
    int *status;
    int box;       // keys of a TMA box
    int slot_dim;  // coordinate (1 or 2) of the slot; the other one is the head
};
struct TcMaps {
    CUtensorMap k, v;
};

__device__ __forceinline__ bool wait_bounded(uint64_t *bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (clock64() - t0 > (1ll << 31)) return false;
    }
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
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
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
__device__ __forceinline__ void tmem_st2(uint32_t addr, float a, float b) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(__float_as_uint(a)), "r"(__float_as_uint(b)) : "memory");
}
__device__ __forceinline__ float2 tmem_ld2(uint32_t addr) {
    uint32_t a, b;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
// f16 weights are held 2^6 larger, which keeps small ones out of the subnormals; at most 2^(6 + 8) < 65504
template <typename T> constexpr float lift() { return std::is_same<T, __half>::value ? 6.f : 0.f; }

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

// Tiles reach shared memory in the order in which the tensor cores take them: K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1)
__device__ __forceinline__ uint32_t k_tile(uint32_t j) { return j ? 2 * j - 1 : 0; }
__device__ __forceinline__ uint32_t v_tile(uint32_t j, uint32_t n) { return j + 1 == n ? 2 * n - 1 : 2 * j + 2; }

template <typename T, int D> __global__ void __launch_bounds__(TT, 1) tree_attn_tc_kernel(const __grid_constant__ TcParams prm, const __grid_constant__ TcMaps maps) {
    using C = Cfg<D>;
    using W = Walk<TM, TK>;
    constexpr int NST = C::STAGES;
    extern __shared__ __align__(1024) uint8_t gsm[];
    uint8_t *const q_sm = (uint8_t *)(((uintptr_t)gsm + 1023) & ~(uintptr_t)1023), *const ring = q_sm + C::ATOMS * TM * 128;
    __shared__ uint64_t full[NST], empty[NST], s_full[2], p_full[2], o_done[2], q_full, x_full, epi_done;
    __shared__ uint32_t tmem_s, odd_sm; // odd_sm: number of the last segment with values set aside
    const TreeDev &p = prm.t;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < NST; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int s = 0; s < 2; ++s) mbar_init(&s_full[s], 1), mbar_init(&p_full[s], 4), mbar_init(&o_done[s], 1);
        mbar_init(&q_full, 8), mbar_init(&x_full, 8), mbar_init(&epi_done, 8);
        mbar_fence_init();
        odd_sm = 0;
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    pdl_wait_prior();
    pdl_launch_dependents();
    const Share share = cta_share<TM, TK, TT, 1>(p); // (its barriers also publish the set-up above)
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_s;
    if (tid == 0) p.meta[blockIdx.x * TREE_META] = make_int4(-1, 0, 0, 0);
    __syncthreads(); // ordered before the record of the CTA's cut unit
    bool ok = true;

    if (warp == 0) {
        // ---- TMA: lane -> (64 values, box of keys) ----
        const int atom = lane % C::ATOMS, part = lane / C::ATOMS, box = prm.box, parts = TK / box;
        const bool mine = part < parts;
        uint32_t tile0 = 0;
        for (W w(p, share); w.more() && ok; w.next()) {
            const int key_end = Tiles<TM, TK>::key_end(p, w.v, w.t), n = w.end - w.blk;
            const int *const table = p.blocks + (size_t)w.v.id * p.max_blocks;
            auto page_of = [&](int j) { // page of this lane's box in block j of the segment
                const int token = (w.blk + j) * TK + part * box;
                return mine && j < n && token < key_end ? table[token / p.page_size] : 0;
            };
            auto load = [&](const CUtensorMap *map, int j, uint32_t tile, int page) {
                const uint32_t st = tile % NST;
                if (tile >= NST && !wait_bounded(&empty[st], (tile / NST - 1) & 1)) return false;
                const int token = (w.blk + j) * TK + part * box;
                const bool go = mine && token < key_end;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, go));
                if (lane == 0) mbar_arrive_expect_tx(&full[st], boxes * box * 128);
                __syncwarp();
                if (go) {
                    const int slot = token % p.page_size;
                    tma_box(smem_u32(ring) + st * C::TILE + atom * (TK * 128) + part * box * 128, map, atom * 64, prm.slot_dim == 1 ? slot : w.h,
                            prm.slot_dim == 1 ? w.h : slot, page, smem_u32(&full[st]));
                }
                return true;
            };
            int prev = 0, cur = page_of(0);
            for (int i = 0; i <= n && ok; ++i) {
                const int next = page_of(i + 1);
                if (i < n) ok = load(&maps.k, i, tile0 + k_tile(i), cur);
                if (i > 0 && ok) ok = load(&maps.v, i - 1, tile0 + v_tile(i - 1, n), prev);
                prev = cur, cur = next;
            }
            tile0 += 2 * n;
        }
    } else if (warp == 1) {
        // ---- MMA issue ----
        uint32_t tile0 = 0, seg = 0, done[2] = {0, 0};
        const uint32_t q0 = smem_u32(q_sm), r0 = smem_u32(ring);
        for (W w(p, share); w.more() && ok; w.next(), ++seg) {
            const uint32_t n = w.end - w.blk;
            ok = wait_bounded(&q_full, seg & 1);
            if (ok && seg) ok = wait_bounded(&epi_done, (seg - 1) & 1); // the accumulators have been read
            for (uint32_t i = 0; i <= n && ok; ++i) {
                if (i < n) {
                    const uint32_t tile = tile0 + k_tile(i), st = tile % NST;
                    if (!(ok = wait_bounded(&full[st], tile / NST & 1))) break;
                    fence_after();
                    if (lane == 0) {
                        // the score tile's last user, P V of the block before last, was issued earlier and runs before
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            const uint32_t off = (kk / 4) * (TK * 128) + (kk % 4) * 32;
                            mma_ss(tmem + (i & 1) * 128, desc_k_major(q0 + off), desc_k_major(r0 + st * C::TILE + off), idesc<T>(TK, false), kk > 0);
                        }
                        mma_commit(&empty[st]);
                        mma_commit(&s_full[i & 1]);
                    }
                    __syncwarp();
                }
                if (i > 0) {
                    const uint32_t j = i - 1, s = j & 1, tile = tile0 + v_tile(j, n), st = tile % NST;
                    if (!(ok = wait_bounded(&full[st], tile / NST & 1) && wait_bounded(&p_full[s], done[s] & 1))) break;
                    fence_after();
                    if (lane == 0) {
#pragma unroll
                        for (int kk = 0; kk < TK / 16; ++kk)
                            mma_ts(tmem + C::O_COL + s * D, tmem + s * 128 + kk * 8, desc_mn_major(r0 + st * C::TILE + kk * 16 * 128), idesc<T>(D, true), j >= 2 || kk > 0);
                        mma_commit(&empty[st]);
                        mma_commit(&o_done[s]);
                    }
                    __syncwarp();
                    ++done[s];
                }
            }
            tile0 += 2 * n;
        }
    } else if (warp >= 4) {
        // ---- the streams ----
        const uint32_t s = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t t_lane = tmem + (quarter * 32u << 16), t_s = t_lane + s * 128, t_o = t_lane + C::O_COL + s * D;
        uint32_t tile0 = 0, seg = 0, done[2] = {0, 0};
        for (W w(p, share); w.more() && ok; w.next(), ++seg) {
            const SeqView v = w.v;
            const uint32_t n = w.end - w.blk;
            const int row0 = w.t * TM, rows = min(TM, v.n * p.group - row0);
            const int key_end = Tiles<TM, TK>::key_end(p, v, w.t);
            { // queries: 16-byte pieces into the swizzled rows
                constexpr int PIECES = D / 8;
                for (int c = tid - 128; c < TM * PIECES; c += 256) {
                    const int r = c / PIECES, d = c % PIECES;
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (r < rows)
                        x = *(const uint4 *)((const T *)p.q + (v.r0 + (row0 + r) / p.group) * p.q_stride + (w.h * p.group + (row0 + r) % p.group) * D + d * 8);
                    *(uint4 *)(q_sm + (d / 8) * (TM * 128) + r * 128 + (((d % 8) ^ (r & 7)) << 4)) = x;
                }
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
            }
            const int me = (row0 + min((int)row, rows - 1)) / p.group; // this row's index in the sequence
            float m = -INFINITY, l = 0.f; // reference (a power of two), sum of weights
            for (uint32_t j = s; j < n && ok; j += 2) {
                const int key0 = (w.blk + j) * TK;
                const bool tail = key0 + TK > v.ctx;
                if (!(ok = wait_bounded(&s_full[s], done[s] & 1))) break;
                fence_after();
                if (tail) { // clean the values of this block: thread = key
                    const uint32_t tile = tile0 + v_tile(j, n), st = tile % NST;
                    if (!(ok = wait_bounded(&full[st], tile / NST & 1))) break;
                    const int token = key0 + (int)(tid & 127);
                    if (token >= v.ctx) {
                        const uint32_t kr = tid & 127;
                        bool odd = false;
#pragma unroll
                        for (int a = 0; a < C::ATOMS; ++a)
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                uint4 *const at = (uint4 *)(ring + st * C::TILE + a * (TK * 128) + kr * 128 + c * 16);
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
                        if (odd) odd_sm = seg + 1;
                    }
                    fence_async();
                }
                // two passes over the scores, 64 columns in registers at a time: reading tensor memory twice costs less
                // than what 128 live values spill
                uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
                if (tail)
#pragma unroll
                    for (int c = 0; c < 4; ++c) bits[c] = view_bits(p, v, me, key0 + 32 * c);
                auto scores = [&](int half, uint32_t(&x)[64]) {
                    tmem_ld32(t_s + 64 * half, x);
                    tmem_ld32(t_s + 64 * half + 32, x + 32);
                    wait_ld();
                    if (tail)
#pragma unroll
                        for (int e = 0; e < 64; ++e)
                            if (!(bits[2 * half + e / 32] >> (e % 32) & 1u)) x[e] = 0xff800000u;
                };
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t x[64];
                    scores(half, x);
#pragma unroll
                    for (int e = 0; e < 64; ++e) top[e & 3] = fmaxf(top[e & 3], __uint_as_float(x[e]));
                }
                const float block_max = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2 - lift<T>();
                if (__any_sync(0xffffffffu, block_max > m + 8.f)) {
                    const float to = block_max > m + 8.f ? block_max : m;
                    const float corr = m == to ? 1.f : ex2(m - to);
                    if (j >= 2) {
                        if (!(ok = wait_bounded(&o_done[s], (done[s] - 1) & 1))) break; // P V of the stream's block before
                        fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(t_o + c, o);
                            wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                            tmem_st32(t_o + c, o);
                        }
                    }
                    l *= corr, m = to;
                }
                const float sub = m == -INFINITY ? 0.f : m; // nothing seen yet: every weight is 2^-inf
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t x[64];
                    scores(half, x);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w16[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float a = ex2(fmaf(__uint_as_float(x[32 * c + 2 * e]), p.scale_log2, -sub));
                            const float b = ex2(fmaf(__uint_as_float(x[32 * c + 2 * e + 1]), p.scale_log2, -sub));
                            sum[e & 1] += a, sum[2 + (e & 1)] += b;
                            w16[e] = pack2<T>(a, b);
                        }
                        tmem_st16(t_s + 32 * half + 16 * c, w16);
                    }
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[s]);
                ++done[s];
            }
            if (!ok) break;
            // ---- join the streams' parts, store ----
            done[1 - s] += s == 0 ? n / 2 : (n + 1) / 2;
            tmem_st2(t_s + 64, m, l); // behind the weights, in columns that only scores use
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&x_full);
            ok = wait_bounded(&x_full, seg & 1) && wait_bounded(&o_done[0], (done[0] - 1) & 1) && (n < 2 || wait_bounded(&o_done[1], (done[1] - 1) & 1));
            if (!ok) break;
            fence_after();
            const float2 a = tmem_ld2(t_lane + 64), b1 = tmem_ld2(t_lane + 128 + 64);
            wait_ld();
            const float2 b = n < 2 ? make_float2(-INFINITY, 0.f) : b1;
            const float mm = fmaxf(a.x, b.x);
            const float wa = a.x == -INFINITY ? 0.f : exp2f(a.x - mm), wb = b.x == -INFINITY ? 0.f : exp2f(b.x - mm);
            const float ll = a.y * wa + b.y * wb;
            const bool whole = w.whole(), live = (int)row < rows, odd = odd_sm == seg + 1;
            float *const mine = part_of<TM>(p, blockIdx.x, w.slot());
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
            T *const out = (T *)p.out + (v.r0 + (row0 + row) / p.group) * p.out_stride + (w.h * p.group + (row0 + row) % p.group) * (long long)D;
#pragma unroll
            for (int c = (int)s * (D / 2), u = 0; u < D / 2; u += 32) {
                uint32_t o0[32], o1[32];
                tmem_ld32(t_lane + C::O_COL + c + u, o0);
                tmem_ld32(t_lane + C::O_COL + D + c + u, o1);
                wait_ld();
                float o[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(o0[e]) * wa + (n < 2 ? 0.f : __uint_as_float(o1[e]) * wb);
                if (odd && live) { // infinities and NaN of the tokens that the row sees
                    const int *const table = p.blocks + (size_t)v.id * p.max_blocks;
                    for (int token = max(v.ctx, w.blk * TK); token < min(key_end, w.end * TK); ++token) {
                        const int page = table[token / p.page_size];
                        if ((unsigned)page >= (unsigned)p.n_pages || !sees(p, v, me, token - v.ctx)) continue;
                        const T *const at = (const T *)p.v + page * p.page_stride + token % p.page_size * p.slot_stride + w.h * p.head_stride + c + u;
#pragma unroll 1
                        for (int e4 = 0; e4 < 32; e4 += 4) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) // (a register array wants constant indices)
                                if ((e & ~3) == e4) {
                                    const float y = (float)at[e];
                                    if (!isfinite(y)) o[e] += y;
                                }
                        }
                    }
                }
                if (!live) continue;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[k] = pack2<T>(ll == 0.f ? 0.f : o[e + 2 * k] * inv, ll == 0.f ? 0.f : o[e + 2 * k + 1] * inv);
                        *(uint4 *)(out + c + u + e) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *(float4 *)(mine + (size_t)row * D + c + u + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if (!whole) {
                if (s == 0 && live) *(float2 *)(mine + (size_t)TM * D + 2 * row) = make_float2(mm, ll);
                if (tid == 128 && w.first()) w.record(p.meta + blockIdx.x * TREE_META);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&epi_done);
            tile0 += 2 * n;
        }
    }
    if (!ok) *(volatile int *)prm.status = DEV_TIMEOUT;
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

template <typename T, int D> cudaError_t launch(const DeviceInfo &dev, const TcParams &prm, const TcMaps &maps, bool pdl, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(tree_attn_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
    if (e != cudaSuccess) return e;
    if ((e = launch_kernel(tree_attn_tc_kernel<T, D>, dim3(dev.sm_count), dim3(TT), Cfg<D>::SMEM, st, pdl, prm, maps)) != cudaSuccess) return e;
    return launch_kernel(tree_join_kernel<T, TM>, dim3(dev.sm_count, TM / 8), dim3(256), 0, st, pdl, prm.t);
}

} // namespace

bool tree_attn_tc_supported(const PoolDev &pool, int dtype) {
    if (dtype == ULLM_DTYPE_F32 || pool.elem_bytes != 2 || (pool.head_dim != 64 && pool.head_dim != 128)) return false;
    const int ps = pool.page_size; // a box of keys starts on a swizzle group of eight rows and lies in one page
    return ps % 128 == 0 || ps == 8 || ps == 16 || ps == 32 || ps == 64;
}
size_t tree_attn_tc_work(int sm_count, int dim) { return sizeof(float) * (size_t)sm_count * 2 * TM * (dim + 2); }

cudaError_t launch_tree_attn_tc(const DeviceInfo &dev, const PoolDev &pool, int dtype, const TreeDev &t, int *d_status, bool pdl, cudaStream_t st) {
    TcParams prm;
    TcMaps maps;
    prm.t = t, prm.status = d_status, prm.box = pool.page_size < TK ? pool.page_size : TK, prm.slot_dim = 1;
    if (!encode_pool(pool, dtype, t.k, prm.box, &prm.slot_dim, &maps.k) || !encode_pool(pool, dtype, t.v, prm.box, &prm.slot_dim, &maps.v))
        return cudaErrorNotSupported;
    if (dtype == ULLM_DTYPE_F16) return pool.head_dim == 64 ? launch<__half, 64>(dev, prm, maps, pdl, st) : launch<__half, 128>(dev, prm, maps, pdl, st);
    return pool.head_dim == 64 ? launch<__nv_bfloat16, 64>(dev, prm, maps, pdl, st) : launch<__nv_bfloat16, 128>(dev, prm, maps, pdl, st);
}

} // namespace ullm
