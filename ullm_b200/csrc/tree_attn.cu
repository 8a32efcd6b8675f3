// Attention of drafted rows over a paged cache: the kernel for every type, head size and page size, and the entry points.
//
//   o_i = sum_j p_ij v_j,  p_ij = 2^(s_ij - m_i) / sum_k 2^(s_ik - m_i),  s_ij = scale log2(e) q_i . k_j
//
// over the keys that row i sees, in one pass with a running maximum m, sum l and weighted sum of values, all f32.
//
// tree_attn_fma_kernel: f32 arithmetic on the CUDA cores, for f32 queries and for whatever the tensor-core kernel
// (tree_attn_tc.cu) does not take.  A CTA of 256 threads holds 16 query rows and walks blocks of 64 keys that it has
// widened to f32 in shared memory.
#include "engine.h"
#include "tree_sched.cuh"

#include <algorithm>
#include <cmath>

namespace ullm {

constexpr int FM = 16, FK = 64, FT = 256; // rows, keys of a block, threads
constexpr int F_COST = 1, F_MIN = 2;       // places that a unit costs beside its blocks; places that a CTA takes at least

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&o)[8]);
template <> __device__ __forceinline__ void load8<float>(const float *p, float (&o)[8]) {
    const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
    o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__half>(const __half *p, float (&o)[8]) {
    const uint4 v = *(const uint4 *)p;
    const __half2 *h = (const __half2 *)&v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        o[2 * i] = f.x, o[2 * i + 1] = f.y;
    }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&o)[8]) {
    const uint4 v = *(const uint4 *)p;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) o[2 * i] = __uint_as_float(w[i] << 16), o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}

constexpr int fma_kp(int dim) { return dim + 4; } // padded key row: 128-bit reads one row apart hit distinct banks
constexpr int FSP = FM + 4;                        // padded row of the transposed scores
inline size_t fma_smem(int dim) { return sizeof(float) * ((size_t)FM * dim + (size_t)FK * fma_kp(dim) + (size_t)FK * dim + FK * FSP + 3 * FM); }

template <typename Q, typename KV> __global__ void __launch_bounds__(FT) tree_attn_fma_kernel(const TreeDev p) {
    extern __shared__ __align__(16) float sm[];
    const int D = p.dim, KP = fma_kp(D), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float *const qs = sm, *const ks = qs + FM * D, *const vs = ks + FK * KP, *const sc = vs + FK * D, *const ms = sc + FK * FSP, *const ls = ms + FM,
                *const cs = ls + FM;
    __shared__ Seg seg;
    pdl_wait_prior();
    pdl_launch_dependents();
    Sched<FM, FK, F_COST, F_MIN> sched(p);
    bool some = false;
    if (warp == 0) {
        if (lane == 0) p.meta[blockIdx.x * TREE_META] = make_int4(-1, 0, 0, 0);
        __syncwarp();
        some = sched.init();
    }
    // weighted sum of values: thread (key part, four rows, four values)
    const int quads = D / 4, per = 4 * quads, split = per <= 64 ? 4 : (per <= 128 ? 2 : 1);
    const int part = tid / per, item = tid % per, rg = item / quads, dq = item % quads;
    const bool pv = part < split;
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
        auto token_of = [&](int r) { return (w.row0 + r) / p.group; };
        auto head_of = [&](int r) { return w.h * p.group + (w.row0 + r) % p.group; };
        for (int i = tid; i < FM * D / 8; i += FT) {
            const int r = i / (D / 8), d = i % (D / 8) * 8;
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (r < rows) load8<Q>((const Q *)p.q + (v.r0 + token_of(r)) * p.q_stride + (long long)head_of(r) * D + d, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) qs[r * D + d + e] = x[e];
        }
        if (tid < FM) ms[tid] = -INFINITY, ls[tid] = 0.f;
        float acc[4][4];
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][e] = 0.f;
        const int *const table = p.blocks + (size_t)v.id * p.max_blocks;
        for (int blk = w.blk; blk < blk_end; ++blk) {
            const int k0 = blk * FK;
            __syncthreads();
            for (int i = tid; i < FK * D / 8; i += FT) {
                const int j = i / (D / 8), d = i % (D / 8) * 8, token = k0 + j;
                float kk[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, vv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (token < key_end) {
                    const int page = table[token / p.page_size];
                    if ((unsigned)page < (unsigned)p.n_pages) {
                        const long long at = page * p.page_stride + token % p.page_size * p.slot_stride + w.h * p.head_stride + d;
                        load8<KV>((const KV *)p.k + at, kk);
                        load8<KV>((const KV *)p.v + at, vv);
                    }
                    if (token >= v.ctx) { // some rows may not see it: 0 * inf must not reach them
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (!isfinite(vv[e])) vv[e] = 0.f, seg.odd = 1;
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) ks[j * KP + d + e] = kk[e], vs[j * D + d + e] = vv[e];
            }
            __syncthreads();
            { // scores: thread (key, four rows)
                const int j = tid % FK, r0 = tid / FK * 4;
                if (r0 < rows) {
                    float s[4] = {0.f, 0.f, 0.f, 0.f};
                    for (int d = 0; d < D; d += 4) {
                        const float4 k = *(const float4 *)(ks + j * KP + d);
#pragma unroll
                        for (int a = 0; a < 4; ++a) {
                            const float4 q = *(const float4 *)(qs + (r0 + a) * D + d);
                            s[a] += q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
                        }
                    }
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        bool see = k0 + j < key_end && r0 + a < rows;
                        if (see && k0 + j >= v.ctx) see = sees(p, v, token_of(r0 + a), k0 + j - v.ctx);
                        sc[j * FSP + r0 + a] = see ? s[a] * p.scale_log2 : -INFINITY;
                    }
                }
            }
            __syncthreads();
            for (int r = warp; r < rows; r += FT / 32) {
                const float s0 = sc[lane * FSP + r], s1 = sc[(lane + 32) * FSP + r], m = ms[r];
                const float mn = fmaxf(m, warp_max(fmaxf(s0, s1)));
                // nothing seen so far: all weights are zero.  (A score of +inf or NaN gives NaN, as the formula does.)
                const float p0 = s0 == -INFINITY ? 0.f : exp2f(s0 - mn), p1 = s1 == -INFINITY ? 0.f : exp2f(s1 - mn);
                const float corr = m == -INFINITY ? 0.f : exp2f(m - mn), sum = warp_sum(p0 + p1);
                sc[lane * FSP + r] = p0, sc[(lane + 32) * FSP + r] = p1;
                __syncwarp();
                if (lane == 0) ms[r] = mn, ls[r] = ls[r] * corr + sum, cs[r] = corr;
            }
            __syncthreads();
            if (pv && rg * 4 < rows) {
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const float corr = rg * 4 + a < rows ? cs[rg * 4 + a] : 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][e] *= corr;
                }
                const int j0 = part * (FK / split), j1 = j0 + FK / split;
                for (int j = j0; j < j1; ++j) {
                    const float4 x = *(const float4 *)(vs + j * D + dq * 4), q = *(const float4 *)(sc + j * FSP + rg * 4);
                    const float xs[4] = {x.x, x.y, x.z, x.w}, qq[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int a = 0; a < 4; ++a)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[a][e] += qq[a] * xs[e];
                }
            }
        }
        __syncthreads();
        // sum the key parts in order, in the keys' memory
        float *const red = ks;
        if (pv)
#pragma unroll
            for (int a = 0; a < 4; ++a)
                if (rg * 4 + a < rows) *(float4 *)(red + ((size_t)part * FM + rg * 4 + a) * D + dq * 4) = make_float4(acc[a][0], acc[a][1], acc[a][2], acc[a][3]);
        __syncthreads();
        const bool whole = w.flags & 1, odd = seg.odd;
        float *const mine = whole ? nullptr : part_of<FM>(p, blockIdx.x, w.flags >> 1);
        for (int i = tid; i < rows * D; i += FT) {
            const int r = i / D, d = i % D;
            float o = 0.f;
            for (int s = 0; s < split; ++s) o += red[((size_t)s * FM + r) * D + d];
            if (odd) { // infinities and NaN of the tokens that the row does see
                const int first = max(v.ctx, w.blk * FK), last = min(key_end, blk_end * FK), me = token_of(r);
                for (int token = first; token < last; ++token) {
                    const int page = table[token / p.page_size];
                    if ((unsigned)page >= (unsigned)p.n_pages || !sees(p, v, me, token - v.ctx)) continue;
                    const long long at = page * p.page_stride + token % p.page_size * p.slot_stride + w.h * p.head_stride + d;
                    const float x = (float)((const KV *)p.v)[at];
                    if (!isfinite(x)) o += x;
                }
            }
            if (whole) {
                const float l = ls[r];
                ((Q *)p.out)[(v.r0 + token_of(r)) * p.out_stride + (long long)head_of(r) * D + d] = out_from<Q>(l == 0.f ? 0.f : o / l);
            } else {
                mine[i] = o;
            }
        }
        if (!whole && tid < rows) *(float2 *)(mine + (size_t)FM * D + 2 * tid) = make_float2(ms[tid], ls[tid]);
    }
}

// CTAs of the f32 kernel: as many as the SMs hold at once
static int fma_ctas(int sm_count, int dim) { return sm_count * (dim <= 64 ? 4 : (dim <= 128 ? 2 : 1)); }
static size_t meta_bytes(int ctas) { return ((size_t)ctas * TREE_META * sizeof(int4) + 255) / 256 * 256; }

template <typename Q, typename KV> static cudaError_t launch_fma(const DeviceInfo &dev, const TreeDev &t, bool pdl, cudaStream_t st) {
    const size_t smem = fma_smem(t.dim);
    cudaError_t e = cudaFuncSetAttribute(tree_attn_fma_kernel<Q, KV>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fma_smem(256));
    if (e != cudaSuccess) return e;
    const int ctas = fma_ctas(dev.sm_count, t.dim);
    e = launch_kernel(tree_attn_fma_kernel<Q, KV>, dim3(ctas), dim3(FT), smem, st, pdl, t);
    if (e != cudaSuccess) return e;
    return launch_kernel(tree_join_kernel<Q, FM>, dim3(dev.sm_count * JOIN_PER_SM), dim3(32 * JOIN_WARPS), 0, st, pdl, t, ctas);
}

} // namespace ullm

using namespace ullm;

static size_t tree_work_bytes(int sm_count, int dim, bool tc) {
    const int ctas = fma_ctas(sm_count, dim);
    const size_t fma = sizeof(float) * (size_t)ctas * 2 * FM * (dim + 2);
    return meta_bytes(ctas) + (tc ? std::max(fma, tree_attn_tc_work(sm_count, dim)) : fma);
}

size_t ullm_cuda_tree_attn_work_bytes(const ullm_cuda_ctx *c, const ullm_kv_pages *kv, int dtype) {
    PoolDev pool;
    if (!c || !kv || pool_check(kv, &pool)) return 0;
    return tree_work_bytes(c->dev.sm_count, pool.head_dim, tree_attn_tc_supported(pool, dtype));
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
    if (!std::isfinite(a->scale) || a->scale < 0.f || (a->scale > 0.f && a->scale < 1e-30f))
        return ctx_fail(c, ULLM_ERR_FORMAT, "scale must be finite, at least 1e-30 or 0 for the default");
    { // the line of all blocks is counted in 32 bits (with what the smaller tiles of the f32 kernel would need)
        const double units = ((double)a->n_rows * (a->n_head / a->kv->n_kv_head) / 16 + (double)a->n_seq) * a->kv->n_kv_head;
        if (units * ((double)a->max_blocks * a->kv->page_size / 64 + 4) > 2147483000.0)
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
    t.n_rows = (int)a->n_rows, t.n_seq = (int)a->n_seq, t.n_head = (int)a->n_head, t.n_kv = pool.n_kv_head, t.group = t.n_head / t.n_kv;
    t.dim = pool.head_dim, t.n_table = (int)a->n_table, t.max_blocks = (int)a->max_blocks, t.n_pages = pool.n_pages, t.page_size = pool.page_size;
    t.mask_words = (int)a->mask_words, t.layer = (int)a->layer;
    t.scale_log2 = (float)((a->scale == 0.f ? 1.0 / std::sqrt((double)dim) : (double)a->scale) * 1.4426950408889634);
    DeviceGuard guard(c->device);
    const cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    t.meta = (int4 *)a->d_work, t.part = (float *)((uint8_t *)a->d_work + meta_bytes(fma_ctas(c->dev.sm_count, t.dim)));
    cudaError_t e = cudaErrorNotSupported;
    if (tree_attn_tc_supported(pool, a->dtype)) e = launch_tree_attn_tc(c->dev, pool, a->dtype, t, c->d_status, c->use_pdl, st);
    if (e != cudaErrorNotSupported) { // (strides that a tensor map cannot describe go to the f32 kernel)
        ULLM_CUDA_TRY(c, e);
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
