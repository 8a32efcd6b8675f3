// Attention of drafted rows over a paged cache: the kernel for every type, head size and page size, and the entry points.
//
//   o_i = sum_j p_ij v_j,  p_ij = 2^(s_ij - m_i) / sum_k 2^(s_ik - m_i),  s_ij = scale log2(e) q_i . k_j
//
// over the keys that row i sees, in one pass with a running maximum m, sum l and weighted sum of values, all f32.
//
// tree_attn_fma_kernel: f32 arithmetic on the CUDA cores, for the head sizes, page sizes and strides that the kernels on the tensor cores do not take
// (tree_attn_tc.cu: 16-bit queries; tree_attn_split.cu: f32 queries, heads of 64 and 128).
// A CTA of 256 threads holds 8 to 32 query rows in shared memory and walks blocks of keys; the next block's keys and values arrive by cp.async, as they lie
// in the pages, while one is worked on.  A warp's scores form a tile, a thread's one of up to 2 keys x 4 rows, so that lanes share what they read from
// shared memory: with a key per lane these reads took three times as long as the multiply-adds, which go two to an instruction.
// Shared memory bounds it all the same: 32 lanes x 16 bytes take four cycles, six such reads feed a tile's 32 multiply-adds per lane, which need eight.
// 90 rows of each of 16 sequences over heads of 96 in 32 bits: 402 us, 16.6 TFLOP/s of the 72 of the f32 units.
#include "engine.h"
#include "tree_sched.cuh"

#include <algorithm>
#include <cmath>

namespace ullm {

constexpr int FT = 256;              // threads
constexpr int F_COST = 1, F_MIN = 2; // places that a unit costs beside its blocks; places that a CTA takes at least
constexpr int F_STATIC = 1280;       // bytes of static shared memory at most
constexpr int F_PER_SM = 2;          // CTAs on an SM at most: 128 registers a thread
constexpr int F_PAD = 16;            // bytes behind a key's row: 128-bit reads one row apart hit distinct banks
constexpr int FSP = 4;               // floats behind a row of queries and of scores, for the same

// Two multiply-adds in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b), "l"(*(unsigned long long *)&c));
    return *(float2 *)&r;
}

// bytes of shared memory: queries, two stages of keys (padded) and values, scores, three numbers per row
inline size_t fma_smem(int dim, int kv_bytes, int rows, int keys) {
    return sizeof(float) * ((size_t)rows * (dim + FSP) + (size_t)rows * (keys + FSP) + 3 * rows) + 2 * (size_t)keys * (2 * dim * kv_bytes + F_PAD);
}

template <typename Q, typename KV, int M, int KEYS> __global__ void __launch_bounds__(FT, F_PER_SM) tree_attn_fma_kernel(const TreeDev p) {
    extern __shared__ __align__(16) uint8_t fsm[];
    constexpr int SP = KEYS + FSP, KS = KEYS / 32, RW = M / (FT / 32); // RW: rows of a warp
    // A thread's scores: KT keys x R rows; its weighted sums: PR rows x four values, U times
    constexpr int KT = M == 8 ? 1 : 2, TILES = KEYS / (8 * KT), GROUPS = FT / 32 / TILES, R = M / GROUPS / 4;
    constexpr int PR = 4, U = M == 32 ? 2 : 1;
    const int D = p.dim, QP = D + FSP, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row_b = D * (int)sizeof(KV), key_b = row_b + F_PAD;
    float *const qs = (float *)fsm, *const sc = qs + M * QP, *const ms = sc + M * SP, *const ls = ms + M, *const cs = ls + M;
    uint8_t *const stage0 = (uint8_t *)(cs + M);
    const int stage_b = KEYS * (key_b + row_b);
    __shared__ Seg seg;
    __shared__ long long offs[2][KEYS]; // where the keys of a block lie: bytes behind p.k and p.v, -1 for none
    pdl_wait_prior();
    pdl_launch_dependents();
    Sched<M, KEYS, F_COST, F_MIN> sched(p);
    bool some = false;
    if (warp == 0) {
        if (lane == 0) p.meta[blockIdx.x * TREE_META] = make_int4(-1, 0, 0, 0);
        __syncwarp();
        some = sched.init();
    }
    const int quads = D / 4;
    // pieces of a row; a thread's first piece of a block, and how far it is to its next one
    const int pieces = row_b / 16, step_j = FT / pieces, step_c = FT % pieces, first_j = tid / pieces, first_c = tid % pieces;
    for (;;) {
        __syncthreads();
        if (warp == 0) {
            Seg next;
            next.count = 0;
            if (some) next = sched.next(p.meta + blockIdx.x * TREE_META);
            if (lane == 0) seg = next;
        }
        __syncthreads();
        const Seg w = seg;
        if (!w.count) break;
        SeqView v;
        v.r0 = w.r0, v.n = w.n, v.id = w.id, v.ctx = w.ctx, v.kv = w.kv;
        const int rows = w.rows, key_end = w.key_end, blk_end = w.blk + w.count;
        // weighted sums of values: items (PR rows, four values), spread over the threads, each for a part of the keys
        const int items = (rows + PR - 1) / PR * quads;
        int split = 1;
        while (split * items * 2 <= FT && split * 8 <= KEYS && split * rows * D * (int)sizeof(float) <= stage_b) split *= 2; // (they meet in the stages' memory)
        const int part = split > 1 ? tid / items : 0, item0 = split > 1 ? tid % items : tid;
        auto token_of = [&](int r) { return (w.row0 + r) / p.group; };
        auto head_of = [&](int r) { return w.h * p.group + (w.row0 + r) % p.group; };
        const int *const table = p.blocks + (size_t)v.id * p.max_blocks;
        auto page_at = [&](int token) { return token < key_end ? table[token / p.page_size] : -1; };
        auto place = [&](int page, int token) { // a key behind the last, or of a page outside the pool, has none
            return (unsigned)page < (unsigned)p.n_pages ? (page * p.page_stride + token % p.page_size * p.slot_stride + w.h * p.head_stride) * (long long)sizeof(KV) : -1ll;
        };
        // 16-byte pieces of a block's keys and values; zeros for a key that has no place
        auto fetch = [&](int blk, uint8_t *stage) {
            const long long *const at = offs[(blk - w.blk) & 1];
            int j = first_j, c = first_c;
#pragma unroll 2
            while (j < KEYS) {
                const long long off = at[j];
                const bool on = off >= 0;
                const long long from = on ? off + c * 16 : 0;
                copy16(stage + j * key_b + c * 16, p.k + from, on);
                copy16(stage + KEYS * key_b + j * row_b + c * 16, p.v + from, on);
                j += step_j, c += step_c;
                if (c >= pieces) c -= pieces, ++j;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        if (tid < 2 * KEYS) { // the first two blocks' keys, one per thread
            const int token = w.blk * KEYS + tid;
            offs[tid / KEYS][tid % KEYS] = place(page_at(token), token);
        }
        __syncthreads();
        fetch(w.blk, stage0);
        for (int i = tid; i < M * quads; i += FT) {
            const int r = i / quads, d = i % quads * 4;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) x = widen4((const Q *)p.q + (v.r0 + token_of(r)) * p.q_stride + (long long)head_of(r) * D + d);
            *(float4 *)(qs + r * QP + d) = x;
        }
        // a warp's rows are every eighth: the reference of each, and the lane's share of its sum
        float m_r[RW], l_r[RW];
#pragma unroll
        for (int a = 0; a < RW; ++a) m_r[a] = -INFINITY, l_r[a] = 0.f;
        float2 acc[U][PR][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int a = 0; a < PR; ++a) acc[u][a][0] = acc[u][a][1] = make_float2(0.f, 0.f);
        for (int blk = w.blk; blk < blk_end; ++blk) {
            uint8_t *const stage = stage0 + ((blk - w.blk) & 1) * stage_b;
            const KV *const vs = (const KV *)(stage + KEYS * key_b);
            const int k0 = blk * KEYS;
            if (blk + 1 < blk_end) {
                fetch(blk + 1, stage0 + ((blk + 1 - w.blk) & 1) * stage_b);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncthreads();
            // the block after the next: its page numbers travel while the scores are made
            const int ahead = (blk + 2) * KEYS + tid;
            const bool more = tid < KEYS && blk + 2 < blk_end;
            const int page = more ? page_at(ahead) : -1;
            if (k0 + KEYS > v.ctx) { // the rows' own tokens: some rows may not see them, and 0 * inf must not reach those
                KV *const own = (KV *)(stage + KEYS * key_b);
                for (int i = max(v.ctx - k0, 0) * D + tid; i < min(key_end - k0, KEYS) * D; i += FT)
                    if (!isfinite((float)own[i])) own[i] = (KV)0.f, seg.odd = 1;
            }
            { // scores: warps (tile of keys, tile of rows), lanes 8 x 4, a thread every eighth of its keys and every fourth of its rows
                const int j0 = warp % TILES * (8 * KT) + lane % 8, r0 = warp / TILES * (4 * R) + lane / 8;
                if (warp / TILES * (4 * R) < rows) {
                    float2 s[KT][R]; // sums over the even and the odd values of a head
#pragma unroll
                    for (int b = 0; b < KT; ++b)
#pragma unroll
                        for (int a = 0; a < R; ++a) s[b][a] = make_float2(0.f, 0.f);
                    const uint8_t *const key = stage + j0 * key_b;
#pragma unroll 4
                    for (int d = 0; d < D; d += 4) {
                        float4 x[KT];
#pragma unroll
                        for (int b = 0; b < KT; ++b) x[b] = widen4((const KV *)(key + 8 * b * key_b) + d);
#pragma unroll
                        for (int a = 0; a < R; ++a) {
                            const float4 q = *(const float4 *)(qs + (r0 + 4 * a) * QP + d);
#pragma unroll
                            for (int b = 0; b < KT; ++b) {
                                s[b][a] = fma2(make_float2(q.x, q.y), make_float2(x[b].x, x[b].y), s[b][a]);
                                s[b][a] = fma2(make_float2(q.z, q.w), make_float2(x[b].z, x[b].w), s[b][a]);
                            }
                        }
                    }
#pragma unroll
                    for (int a = 0; a < R; ++a)
#pragma unroll
                        for (int b = 0; b < KT; ++b) {
                            const int r = r0 + 4 * a, j = j0 + 8 * b;
                            bool see = k0 + j < key_end && r < rows;
                            if (see && k0 + j >= v.ctx) see = sees(p, v, token_of(r), k0 + j - v.ctx);
                            sc[r * SP + j] = see ? (s[b][a].x + s[b][a].y) * p.scale_log2 : -INFINITY;
                        }
                }
            }
            __syncthreads();
            if (more) offs[(blk - w.blk) & 1][tid] = place(page, ahead);
            float s[RW][KS], mn[RW];
#pragma unroll
            for (int a = 0; a < RW; ++a) {
                mn[a] = -INFINITY;
                if (a * (FT / 32) < rows) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) s[a][k] = sc[(warp + a * (FT / 32)) * SP + lane + 32 * k], mn[a] = fmaxf(mn[a], s[a][k]);
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int a = 0; a < RW; ++a)
                    if (a * (FT / 32) < rows) mn[a] = fmaxf(mn[a], __shfl_xor_sync(0xffffffffu, mn[a], o));
#pragma unroll
            for (int a = 0; a < RW; ++a) { // (what lies behind the last row is worked on and never written)
                if (a * (FT / 32) >= rows) continue;
                const int r = warp + a * (FT / 32);
                mn[a] = fmaxf(m_r[a], mn[a]);
                const float corr = m_r[a] == -INFINITY ? 0.f : exp2f(m_r[a] - mn[a]);
                l_r[a] *= corr, m_r[a] = mn[a];
                // nothing seen so far: all weights are zero.  (A score of +inf or NaN gives NaN, as the formula does.)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const float x = s[a][k] == -INFINITY ? 0.f : exp2f(s[a][k] - mn[a]);
                    l_r[a] += x;
                    sc[r * SP + lane + 32 * k] = x;
                }
                if (lane == 0) cs[r] = corr;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int item = item0 + u * FT, rg = item / quads, dq = item % quads;
                if (part >= split || item >= items) continue;
#pragma unroll
                for (int a = 0; a < PR; ++a) {
                    const float corr = rg * PR + a < rows ? cs[rg * PR + a] : 0.f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) acc[u][a][e].x *= corr, acc[u][a][e].y *= corr;
                }
                const int j0 = part * (KEYS / split), j1 = j0 + KEYS / split;
#pragma unroll 2
                for (int j = j0; j < j1; j += 4) {
                    float4 q[PR];
#pragma unroll
                    for (int a = 0; a < PR; ++a) q[a] = *(const float4 *)(sc + (rg * PR + a) * SP + j);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float4 x = widen4(vs + (j + k) * D + dq * 4);
#pragma unroll
                        for (int a = 0; a < PR; ++a) {
                            const float wa = k == 0 ? q[a].x : (k == 1 ? q[a].y : (k == 2 ? q[a].z : q[a].w));
                            acc[u][a][0] = fma2(make_float2(wa, wa), make_float2(x.x, x.y), acc[u][a][0]);
                            acc[u][a][1] = fma2(make_float2(wa, wa), make_float2(x.z, x.w), acc[u][a][1]);
                        }
                    }
                }
            }
            __syncthreads(); // the stage and the scores are free
        }
#pragma unroll
        for (int a = 0; a < RW; ++a) {
            const float l = warp_sum(l_r[a]);
            if (lane == 0) ms[warp + a * (FT / 32)] = m_r[a], ls[warp + a * (FT / 32)] = l;
        }
        // sum the key parts in order, in the stages' memory
        float *const red = (float *)stage0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int item = item0 + u * FT, rg = item / quads, dq = item % quads;
            if (part >= split || item >= items) continue;
#pragma unroll
            for (int a = 0; a < PR; ++a)
                if (rg * PR + a < rows) *(float4 *)(red + ((size_t)part * rows + rg * PR + a) * D + dq * 4) = make_float4(acc[u][a][0].x, acc[u][a][0].y, acc[u][a][1].x, acc[u][a][1].y);
        }
        __syncthreads();
        const bool whole = w.flags & 1, odd = seg.odd;
        float *const mine = whole ? nullptr : part_of<M>(p, blockIdx.x, w.flags >> 1);
        for (int i = tid; i < rows * quads; i += FT) {
            const int r = i / quads, d = (i - r * quads) * 4;
            float4 o = *(const float4 *)(red + r * D + d);
            for (int s = 1; s < split; ++s) {
                const float4 x = *(const float4 *)(red + ((size_t)s * rows + r) * D + d);
                o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
            }
            // values that are not finite: of the rows' own tokens they were set aside, of those in front they show in the sums (where the sum of weights is NaN, every value is)
            const bool bad = !(isfinite(o.x) && isfinite(o.y) && isfinite(o.z) && isfinite(o.w)) && ls[r] == ls[r];
            if (odd || bad) {
                const int first = bad ? w.blk * KEYS : max(v.ctx, w.blk * KEYS), last = min(key_end, blk_end * KEYS), me = token_of(r);
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int token = first; token < last; ++token) {
                    const int page = table[token / p.page_size];
                    if ((unsigned)page >= (unsigned)p.n_pages || (token >= v.ctx && !sees(p, v, me, token - v.ctx))) continue;
                    const long long at = page * p.page_stride + token % p.page_size * p.slot_stride + w.h * p.head_stride;
                    const float4 x = widen4((const KV *)p.v + at + d);
                    if (isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w)) continue;
                    const bool none = has_no_weight((const Q *)p.q + (v.r0 + me) * p.q_stride + (long long)head_of(r) * D, (const KV *)p.k + at, D, p.scale_log2);
                    if (!isfinite(x.x)) sum.x += none ? NAN : x.x;
                    if (!isfinite(x.y)) sum.y += none ? NAN : x.y;
                    if (!isfinite(x.z)) sum.z += none ? NAN : x.z;
                    if (!isfinite(x.w)) sum.w += none ? NAN : x.w;
                }
                if (sum.x != 0.f) o.x = sum.x;
                if (sum.y != 0.f) o.y = sum.y;
                if (sum.z != 0.f) o.z = sum.z;
                if (sum.w != 0.f) o.w = sum.w;
            }
            if (whole) {
                const float l = ls[r], inv = l == 0.f ? 0.f : 1.0f / l;
                Q *const out = (Q *)p.out + (v.r0 + token_of(r)) * p.out_stride + (long long)head_of(r) * D + d;
                const float y[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = out_from<Q>(l == 0.f ? 0.f : y[e] * inv);
            } else {
                *(float4 *)(mine + (size_t)r * D + d) = o;
            }
        }
        if (!whole && tid < rows) *(float2 *)(mine + (size_t)M * D + 2 * tid) = make_float2(ms[tid], ls[tid]);
    }
}

// CTAs of the f32 kernel: as many as the SMs hold at once
static int fma_ctas(const DeviceInfo &dev, int dim, int kv_bytes, int rows, int keys) {
    const size_t one = fma_smem(dim, kv_bytes, rows, keys) + 1024 + F_STATIC; // with what the system and the static variables take
    return dev.sm_count * (int)std::max((size_t)1, std::min((size_t)F_PER_SM, (size_t)dev.max_smem_sm / one));
}
static size_t meta_bytes(int ctas) { return ((size_t)ctas * TREE_META * sizeof(int4) + 255) / 256 * 256; }
// Keys of a block: 64 while two CTAs with two stages of them fit an SM, else 32 (32 rows over 16-bit heads of 256, 512 bytes: 194 us with 64 keys and one CTA, 180 with 32 and two).
inline int fma_keys(int row_bytes) { return row_bytes <= 256 ? 64 : 32; }
template <typename Q, typename KV, int M, int KEYS> static cudaError_t launch_fma_as(const DeviceInfo &dev, const TreeDev &t, bool pdl, cudaStream_t st) {
    const size_t smem = fma_smem(t.dim, sizeof(KV), M, KEYS);
    cudaError_t e = cudaFuncSetAttribute(tree_attn_fma_kernel<Q, KV, M, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, dev.max_smem_optin - F_STATIC);
    if (e != cudaSuccess) return e;
    const int ctas = fma_ctas(dev, t.dim, sizeof(KV), M, KEYS);
    e = launch_kernel(tree_attn_fma_kernel<Q, KV, M, KEYS>, dim3(ctas), dim3(FT), smem, st, pdl, t);
    if (e != cudaSuccess) return e;
    return launch_kernel(tree_join_kernel<Q, M>, dim3(dev.sm_count * JOIN_PER_SM<M>), dim3(32 * JOIN_WARPS), 0, st, pdl, t, ctas);
}
template <typename Q, typename KV> static cudaError_t launch_fma(const DeviceInfo &dev, const TreeDev &t, bool pdl, cudaStream_t st) {
    // Rows per sequence and key head, on average.  A tile with room for many more rows than there are leaves threads idle (four rows over heads of 96 in 32 bits: 37.5 us
    // with tiles of 8 rows, 39.6 with 16; in 16 bits 31.2 and 32.7), a smaller one reads the keys more often.
    const long long rows = ((long long)t.n_rows * t.group + t.n_seq - 1) / t.n_seq;
    const bool k64 = fma_keys(t.dim * (int)sizeof(KV)) == 64;
    if (rows > 16) return k64 ? launch_fma_as<Q, KV, 32, 64>(dev, t, pdl, st) : launch_fma_as<Q, KV, 32, 32>(dev, t, pdl, st);
    if (rows > 8) return k64 ? launch_fma_as<Q, KV, 16, 64>(dev, t, pdl, st) : launch_fma_as<Q, KV, 16, 32>(dev, t, pdl, st);
    return k64 ? launch_fma_as<Q, KV, 8, 64>(dev, t, pdl, st) : launch_fma_as<Q, KV, 8, 32>(dev, t, pdl, st);
}

} // namespace ullm

using namespace ullm;

// The work area begins with the CTAs' records and their counters (for the most CTAs of any kernel), then the partial results.
static size_t tree_work_bytes(const DeviceInfo &dev, int dim, bool tc) {
    const size_t fma = sizeof(float) * (size_t)dev.sm_count * F_PER_SM * 2 * 32 * (dim + 2); // of 32 rows, the most that a tile of the f32 kernels has
    return 2 * meta_bytes(dev.sm_count * F_PER_SM) + (tc ? std::max(fma, tree_attn_tc_work(dev.sm_count, dim)) : fma);
}

size_t ullm_cuda_tree_attn_work_bytes(const ullm_cuda_ctx *c, const ullm_kv_pages *kv, int dtype) {
    PoolDev pool;
    if (!c || !kv || pool_check(kv, &pool)) return 0;
    return tree_work_bytes(c->dev, pool.head_dim, tree_attn_tc_supported(pool, dtype));
}

int ullm_cuda_tree_attn_dev(ullm_cuda_ctx *c, const ullm_tree_attn *a, void *stream) {
    if (!c || !a || !a->kv) return ULLM_ERR_INVALID;
    if (a->n_rows && a->n_seq &&
        (!a->kv->d_k || !a->kv->d_v || !a->d_q || !a->d_out || !a->d_cu || !a->d_len || !a->d_blocks || !a->d_work))
        return ctx_fail(c, ULLM_ERR_INVALID, "null pointer in an attention call");
    PoolDev pool;
    if (const char *m = pool_check(a->kv, &pool)) return ctx_fail(c, ULLM_ERR_FORMAT, "%s", m);
    if (a->dtype != ULLM_DTYPE_F32 && a->dtype != a->kv->dtype)
        return ctx_fail(c, ULLM_ERR_UNSUPPORTED, "queries are f32 or of the pages' type");
    if (a->layer >= a->kv->n_layer) return ctx_fail(c, ULLM_ERR_FORMAT, "layer %zu of a pool of %zu", a->layer, a->kv->n_layer);
    if (!a->n_head || a->n_head > 65535 || a->n_head % a->kv->n_kv_head)
        return ctx_fail(c, ULLM_ERR_FORMAT, "%zu query heads over %zu key heads", a->n_head, a->kv->n_kv_head);
    if (a->n_rows > INT32_MAX / 2 || a->n_seq > INT32_MAX / 2 || a->n_rows * a->n_head > INT32_MAX / 2)
        return ctx_fail(c, ULLM_ERR_FORMAT, "too many rows or sequences for one call");
    if (!a->n_table || a->n_table > INT32_MAX / 2 || !a->max_blocks || a->max_blocks > (size_t)(INT32_MAX / 2) / a->kv->page_size)
        return ctx_fail(c, ULLM_ERR_FORMAT, "bad size of the page table");
    if (!a->d_ids && a->n_seq > a->n_table) return ctx_fail(c, ULLM_ERR_FORMAT, "%zu sequences in a table of %zu rows", a->n_seq, a->n_table);
    if (a->d_mask && (!a->mask_words || a->mask_words > 65536)) return ctx_fail(c, ULLM_ERR_FORMAT, "a mask has 1 to 65536 words per row");
    const size_t dim = a->kv->head_dim, qd = a->n_head * dim, qb = dtype_bytes(a->dtype);
    const size_t qs = a->q_stride ? a->q_stride : qd, os = a->out_stride ? a->out_stride : qd;
    if (qs < qd || os < qd) return ctx_fail(c, ULLM_ERR_FORMAT, "row strides must cover all heads");
    if (qs * qb % 16 || os * qb % 16 || (uintptr_t)a->d_q % 16 || (uintptr_t)a->d_out % 16)
        return ctx_fail(c, ULLM_ERR_FORMAT, "rows must start on 16-byte boundaries");
    if (!ints_aligned(a->d_cu, a->d_len, a->d_ids, a->d_blocks, a->d_mask)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    if (!std::isfinite(a->scale) || a->scale < 0.f || (a->scale > 0.f && a->scale < 1e-30f) || a->scale > 2e38f) // (times log2(e) it is a 32-bit number too)
        return ctx_fail(c, ULLM_ERR_FORMAT, "scale must be 1e-30 to 2e38, or 0 for the default");
    { // the line of all blocks is counted in 32 bits (with what the smaller tiles of the f32 kernel would need)
        const double units = ((double)a->n_rows * (a->n_head / a->kv->n_kv_head) / 8 + (double)a->n_seq) * a->kv->n_kv_head;
        if (units * ((double)a->max_blocks * a->kv->page_size / 32 + 4) > 2147483000.0)
            return ctx_fail(c, ULLM_ERR_FORMAT, "rows times table size too large for one call: split the rows");
    }
    if (!a->n_rows || !a->n_seq) return ULLM_OK;
    const size_t need = ullm_cuda_tree_attn_work_bytes(c, a->kv, a->dtype);
    if (a->work_bytes < need) return ctx_fail(c, ULLM_ERR_FORMAT, "the work area has %zu bytes, %zu are needed", a->work_bytes, need);
    if ((uintptr_t)a->d_work % 16) return ctx_fail(c, ULLM_ERR_FORMAT, "the work area must be 16-byte aligned");
    TreeDev t;
    t.q = (const uint8_t *)a->d_q, t.out = (uint8_t *)a->d_out, t.q_stride = (long long)qs, t.out_stride = (long long)os;
    t.cu = a->d_cu, t.len = a->d_len, t.ids = a->d_ids, t.blocks = a->d_blocks, t.mask = a->d_mask;
    const long long layer = (long long)a->layer * pool.layer_stride * pool.elem_bytes;
    t.k = pool.k + layer, t.v = pool.v + layer;
    t.page_stride = pool.page_stride, t.slot_stride = pool.slot_stride, t.head_stride = pool.head_stride;
    t.n_rows = (int)a->n_rows, t.n_seq = (int)a->n_seq, t.n_kv = pool.n_kv_head, t.group = (int)a->n_head / t.n_kv;
    t.dim = pool.head_dim, t.n_table = (int)a->n_table, t.max_blocks = (int)a->max_blocks, t.n_pages = pool.n_pages, t.page_size = pool.page_size;
    t.mask_words = (int)a->mask_words, t.page_log = -1;
    for (int l = 0; l < 31; ++l)
        if (t.page_size == 1 << l) t.page_log = l;
    t.scale_log2 = (float)((a->scale == 0.f ? 1.0 / std::sqrt((double)dim) : (double)a->scale) * 1.4426950408889634);
    DeviceGuard guard(c->device);
    const cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    const size_t records = meta_bytes(c->dev.sm_count * F_PER_SM);
    t.meta = (int4 *)a->d_work, t.count = (int *)((uint8_t *)a->d_work + records), t.part = (float *)((uint8_t *)a->d_work + 2 * records);
    cudaError_t e = cudaErrorNotSupported;
    if (tree_attn_tc_supported(pool, a->dtype)) e = launch_tree_attn_tc(c->dev, pool, a->dtype, t, c->d_status, c->tree_wait_cycles, c->use_pdl, st);
    if (e != cudaErrorNotSupported) { // (strides that a tensor map cannot describe go to the f32 kernel)
        ULLM_CUDA_TRY(c, e);
        return ULLM_OK;
    }
    if (a->dtype == ULLM_DTYPE_F32 && tree_attn_split_supported(t.dim)) {
        ULLM_CUDA_TRY(c, launch_tree_attn_split(c->dev, a->kv->dtype, t, c->use_pdl, st));
        return ULLM_OK;
    }
    if (a->dtype == ULLM_DTYPE_F16) e = launch_fma<__half, __half>(c->dev, t, c->use_pdl, st);
    else if (a->dtype == ULLM_DTYPE_BF16) e = launch_fma<__nv_bfloat16, __nv_bfloat16>(c->dev, t, c->use_pdl, st);
    else if (a->kv->dtype == ULLM_DTYPE_F32) e = launch_fma<float, float>(c->dev, t, c->use_pdl, st);
    else if (a->kv->dtype == ULLM_DTYPE_F16) e = launch_fma<float, __half>(c->dev, t, c->use_pdl, st);
    else e = launch_fma<float, __nv_bfloat16>(c->dev, t, c->use_pdl, st);
    ULLM_CUDA_TRY(c, e);
    return ULLM_OK;
}
