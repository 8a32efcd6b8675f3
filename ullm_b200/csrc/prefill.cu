// Batched prefill of the resident decode engine: all prompt tokens through every layer in one
// pass (GpuForward::forward_batch, crates/ullm-metal/src/forward.rs:757-909; the CPU meaning is
// forward_llama run for positions 0..s-1, crates/ullm-model/src/lib.rs:807-969).
//
// Per layer: rmsnorm of every token -> [q|k] and v projections as tensor-core GEMMs on the
// quantized weights (gemm.cu) -> RoPE of q and k, K/V written to the cache -> causal
// attention of the s new tokens over the cache -> W_o GEMM + residual -> rmsnorm ->
// [gate|up] GEMM with silu(g)*u in its epilogue -> W_down GEMM + residual (epilogue).  Only the last token goes through
// the final norm and the output projection (a matvec).  Prompts longer than PREFILL_CHUNK
// tokens are processed in chunks; the attention reads earlier chunks from the cache.
//
// Below it: a tree of drafted tokens in one pass (the paged operators over the engine's cache), and the accepted rows kept.
#include "decode.h"
#include "engine.h"
#include "paged.h"

#include <cstring>

#include <cuda_fp16.h>

#include <algorithm>
#include <utility>

namespace ullm {

constexpr size_t PREFILL_CHUNK = 512;

// y[t, :] = x[t, :] * (1 / sqrt(mean(x[t, :]^2) + eps)) * w   (math.rs:82-86), one CTA per token
__global__ void __launch_bounds__(256) rmsnorm_batch_kernel(const float *__restrict__ x, const float *__restrict__ w, float eps,
                                                           int n, float *__restrict__ y) {
    __shared__ float red[8];
    const float *xr = x + (size_t)blockIdx.x * n;
    float *yr = y + (size_t)blockIdx.x * n;
    float ss = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) ss += xr[i] * xr[i];
    ss = warp_sum(ss);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    float tot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) tot += red[i];
    const float inv = 1.0f / sqrtf(tot / (float)n + eps);
    for (int i = threadIdx.x; i < n; i += 256) yr[i] = xr[i] * inv * w[i];
}

template <typename T> __device__ __forceinline__ T kv_from(float v);
template <> __device__ __forceinline__ float kv_from<float>(float v) { return v; }
template <> __device__ __forceinline__ __half kv_from<__half>(float v) { return __float2half_rn(v); }
template <typename T> __device__ __forceinline__ float kv_to(T v);
template <> __device__ __forceinline__ float kv_to<float>(float v) { return v; }
template <> __device__ __forceinline__ float kv_to<__half>(__half v) { return __half2float(v); }

// One head: (+ bias) -> (per-head RMSNorm, math.rs:82-86) -> RoPE on interleaved or rotate-half pairs
// (math.rs:116-162, products and sums unfused), in shared memory, by one warp.  Same steps as the
// decode kernel's prologue (decode.cu), so both paths fill the cache with the same values.
template <int HD>
__device__ __forceinline__ void head_prepare_batch(const float *__restrict__ src, const float *__restrict__ bias,
                                                   const float *__restrict__ norm_w, float eps, const float2 *__restrict__ rp, int neox,
                                                   float *dst, int lane) {
    constexpr int E = HD / 32;
    float v[E], ss = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = lane + 32 * e;
        v[e] = src[d] + (bias ? bias[d] : 0.f);
        ss += v[e] * v[e];
    }
    if (norm_w) {
        ss = warp_sum(ss);
        const float inv = 1.0f / sqrtf(ss / (float)HD + eps);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = v[e] * inv * norm_w[lane + 32 * e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) dst[lane + 32 * e] = v[e];
    __syncwarp();
    for (int j = lane; j < HD / 2; j += 32) {
        const int ia = neox ? j : 2 * j, ib = neox ? j + HD / 2 : 2 * j + 1;
        const float a = dst[ia], b = dst[ib];
        const float2 cs = rp[j];
        dst[ia] = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
        dst[ib] = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
    }
    __syncwarp();
}

struct RopeBatchParams {
    float *qk;            // [s, qd + kvd]: q heads then k heads of every token; q is rewritten in place
    const float *v;       // [s, kvd]
    const float2 *rope;
    void *kc, *vc;        // this layer's cache
    const float *q_bias, *k_bias, *v_bias, *q_norm, *k_norm; // optional
    float eps;
    int pos0, n_head, n_kv_head, neox;
};

// one CTA per token, one warp per head in turn; k and v go to the cache
template <int HD, typename KV_T> __global__ void __launch_bounds__(256) rope_kv_batch_kernel(const RopeBatchParams p) {
    __shared__ float buf[8][HD];
    const int t = blockIdx.x, pos = p.pos0 + t, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int qd = p.n_head * HD, kvd = p.n_kv_head * HD;
    float *row = p.qk + (size_t)t * (qd + kvd);
    const float2 *rp = p.rope + (size_t)pos * (HD / 2);
    KV_T *kc = (KV_T *)p.kc, *vc = (KV_T *)p.vc;
    for (int hh = warp; hh < p.n_head + p.n_kv_head; hh += 8) {
        const bool is_q = hh < p.n_head;
        const int hk = hh - p.n_head;
        const float *bias = is_q ? (p.q_bias ? p.q_bias + (size_t)hh * HD : nullptr) : (p.k_bias ? p.k_bias + (size_t)hk * HD : nullptr);
        head_prepare_batch<HD>(row + (size_t)hh * HD, bias, is_q ? p.q_norm : p.k_norm, p.eps, rp, p.neox, buf[warp], lane);
        for (int d = lane; d < HD; d += 32) {
            if (is_q) row[(size_t)hh * HD + d] = buf[warp][d];
            else kc[(size_t)pos * kvd + (size_t)hk * HD + d] = kv_from<KV_T>(buf[warp][d]);
        }
        __syncwarp();
    }
    for (int i = threadIdx.x; i < kvd; i += 256)
        vc[(size_t)pos * kvd + i] = kv_from<KV_T>(p.v[(size_t)t * kvd + i] + (p.v_bias ? p.v_bias[i] : 0.f));
}

// Eight consecutive cache values of one position -> f32 (one 16- or 32-byte load)
__device__ __forceinline__ void kv_load8(const float *p, float (&o)[8]) {
    const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
    o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
}
__device__ __forceinline__ void kv_load8(const __half *p, float (&o)[8]) {
    const uint4 v = *(const uint4 *)p;
    const __half2 *h = (const __half2 *)&v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        o[2 * i] = f.x, o[2 * i + 1] = f.y;
    }
}

// Causal attention of the chunk's queries over cache positions 0 .. pos0 + t (lib.rs:916-938: scores
// q.k / sqrt(hd), softmax, weighted sum of v).  grid (n_head, ceil(s / 8)), 8 warps: one query per
// warp; keys in blocks of 32 staged in shared memory for the CTA's 8 queries (vector loads from the
// cache, rows padded so that 128-bit reads one row apart hit distinct banks); lane j scores key j of
// the block, the block's probabilities are then broadcast lane by lane for the P.V sum, where every
// lane owns HD / 32 output dimensions.  Running max / sum as in any streaming softmax.
template <int HD, typename KV_T>
__global__ void __launch_bounds__(256) attn_prefill_kernel(const float *__restrict__ qk, const KV_T *__restrict__ kc,
                                                          const KV_T *__restrict__ vc, float *__restrict__ out, int s, int pos0,
                                                          int qd, int kvd, int kvmul, float scale) {
    constexpr int E = HD / 32, KP = HD + 4; // padded K row: 16-byte aligned, 4 banks apart per row
    __shared__ __align__(16) float ks[32][KP];
    __shared__ __align__(16) float vs[32][HD];
    const int h = blockIdx.x, kvh = h / kvmul, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.y * 8 + warp;
    const bool valid = t < s;
    const int qpos = pos0 + (valid ? t : s - 1);
    const int last_q = pos0 + min(s - 1, (int)blockIdx.y * 8 + 7); // the CTA's keys end at its last query
    float q[HD];
    {
        const float4 *qp = (const float4 *)(qk + (size_t)(valid ? t : 0) * (qd + kvd) + (size_t)h * HD);
#pragma unroll
        for (int d = 0; d < HD / 4; ++d) {
            const float4 v = qp[d];
            q[4 * d] = v.x * scale, q[4 * d + 1] = v.y * scale, q[4 * d + 2] = v.z * scale, q[4 * d + 3] = v.w * scale;
        }
    }
    float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int k0 = 0; k0 <= last_q; k0 += 32) {
        __syncthreads(); // the previous block's tiles are no longer read
        for (int i = threadIdx.x; i < 32 * (HD / 8); i += 256) { // 8 values per thread and matrix
            const int j = i / (HD / 8), d = (i % (HD / 8)) * 8, kp = min(k0 + j, last_q);
            float kk[8], vv[8];
            kv_load8(kc + (size_t)kp * kvd + (size_t)kvh * HD + d, kk);
            kv_load8(vc + (size_t)kp * kvd + (size_t)kvh * HD + d, vv);
            *(float4 *)&ks[j][d] = make_float4(kk[0], kk[1], kk[2], kk[3]);
            *(float4 *)&ks[j][d + 4] = make_float4(kk[4], kk[5], kk[6], kk[7]);
            *(float4 *)&vs[j][d] = make_float4(vv[0], vv[1], vv[2], vv[3]);
            *(float4 *)&vs[j][d + 4] = make_float4(vv[4], vv[5], vv[6], vv[7]);
        }
        __syncthreads();
        if (k0 > qpos) continue; // this query's keys are exhausted (other warps of the CTA still need the tiles)
        float sc = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 4; ++d) {
            const float4 kv = *(const float4 *)&ks[lane][4 * d];
            sc += q[4 * d] * kv.x + q[4 * d + 1] * kv.y + q[4 * d + 2] * kv.z + q[4 * d + 3] * kv.w;
        }
        if (k0 + lane > qpos) sc = -INFINITY;
        const float mb = warp_max(sc), mn = fmaxf(m, mb);
        const float pj = expf(sc - mn), corr = expf(m - mn);
        l = l * corr + warp_sum(pj);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= corr;
        m = mn;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            const float pb = __shfl_sync(0xffffffffu, pj, j);
            if constexpr (E == 2) {
                const float2 v2 = *(const float2 *)&vs[j][lane * 2];
                acc[0] += pb * v2.x, acc[1] += pb * v2.y;
            } else {
                const float4 v4 = *(const float4 *)&vs[j][lane * 4];
                acc[0] += pb * v4.x, acc[1] += pb * v4.y, acc[2] += pb * v4.z, acc[3] += pb * v4.w;
            }
        }
    }
    if (valid) {
        const float inv = 1.0f / l;
#pragma unroll
        for (int e = 0; e < E; ++e) out[(size_t)t * qd + (size_t)h * HD + lane * E + e] = acc[e] * inv;
    }
}

bool Forward::batch_supported() const {
    for (const Layer &L : layers) {
        if (!L.qk_fused || !L.gu_fused) return false;
        const size_t qd = P.n_head * P.head_dim, kvd = P.n_kv_head * P.head_dim;
        if (!gemm_tc_supported(L.wqk.fmt, qd + kvd, P.n_embd, 1) || !gemm_tc_supported(L.wv.fmt, kvd, P.n_embd, 1) ||
            !gemm_tc_supported(L.wo.fmt, P.n_embd, qd, 1) || !gemm_tc_supported(L.wgu.fmt, 2 * P.n_ff, P.n_embd, 1) ||
            !gemm_tc_supported(L.wd.fmt, P.n_embd, P.n_ff, 1))
            return false;
    }
    return P.head_dim == 64 || P.head_dim == 128;
}

// Activation buffers for one chunk, allocated on first use.
cudaError_t Forward::batch_buffers() {
    cudaError_t e;
#define TRY(x) \
    if ((e = (x)) != cudaSuccess) return e;
    if (bscratch) return cudaSuccess;
    const size_t hd = P.head_dim, qd = P.n_head * hd, kvd = P.n_kv_head * hd, E = P.n_embd, F = P.n_ff, B = PREFILL_CHUNK;
    size_t scratch = 0;
    for (const auto &d : {std::pair<size_t, size_t>{qd + kvd, E}, {kvd, E}, {E, qd}, {2 * F, E}, {E, F}})
        for (size_t n = 1; n <= B; ++n) // the split-K factor, and with it the partial-sum area, depends on the token count
            scratch = std::max(scratch, gemm_tc_scratch_bytes(d.first, d.second, n, dev.sm_count));
    if (!bx) TRY(dev_alloc((void **)&bx, B * E * 4));
    if (!bxn) TRY(dev_alloc((void **)&bxn, B * std::max(E, qd) * 4));
    if (!bqk) TRY(dev_alloc((void **)&bqk, B * (qd + kvd) * 4));
    if (!bv) TRY(dev_alloc((void **)&bv, B * kvd * 4));
    if (!bh) TRY(dev_alloc((void **)&bh, B * F * 4));
    TRY(dev_alloc(&bscratch, scratch));
#undef TRY
    return cudaSuccess;
}

cudaError_t Forward::forward_batch(const float *embeds_host, size_t s, float *logits_host) {
    cudaError_t e;
#define TRY(x) \
    if ((e = (x)) != cudaSuccess) return e;
    TRY(cudaSetDevice(device));
    if (!batch_supported()) return cudaErrorNotSupported;
    if (s == 0 || s > P.n_ctx) return cudaErrorInvalidValue;
    const size_t hd = P.head_dim, qd = P.n_head * hd, kvd = P.n_kv_head * hd, E = P.n_embd, B = PREFILL_CHUNK;
    const size_t kvb = P.kv_f16 ? 2 : 4;
    TRY(batch_buffers());
    auto gemm = [&](const Mat &m, const float *in, float *out, size_t n, int epi = EPI_STORE, const float *res = nullptr) {
        ++launches;
        return launch_gemm_tc(m.fmt, m.w, in, out, bscratch, m.out, m.cols, n, dev.sm_count, d_status, stream, epi, res);
    };
    const float scale = 1.0f / sqrtf((float)hd);
    for (size_t c0 = 0; c0 < s; c0 += B) {
        const size_t n = std::min(B, s - c0);
        TRY(cudaMemcpyAsync(bx, embeds_host + c0 * E, n * E * 4, cudaMemcpyHostToDevice, stream));
        for (size_t l = 0; l < P.n_layer; ++l) {
            Layer &L = layers[l];
            uint8_t *kc = (uint8_t *)kcache + l * P.n_ctx * kvd * kvb, *vc = (uint8_t *)vcache + l * P.n_ctx * kvd * kvb;
            rmsnorm_batch_kernel<<<(unsigned)n, 256, 0, stream>>>(bx, L.attn_norm, P.eps, (int)E, bxn);
            TRY(gemm(L.wqk, bxn, bqk, n));
            TRY(gemm(L.wv, bxn, bv, n));
            const dim3 ag((unsigned)P.n_head, (unsigned)((n + 7) / 8));
            const int kvmul = (int)(P.n_head / P.n_kv_head);
            RopeBatchParams rb;
            rb.qk = bqk, rb.v = bv, rb.rope = rope, rb.kc = kc, rb.vc = vc;
            rb.q_bias = L.q_bias, rb.k_bias = L.k_bias, rb.v_bias = L.v_bias, rb.q_norm = L.q_norm, rb.k_norm = L.k_norm;
            rb.eps = P.eps, rb.pos0 = (int)c0, rb.n_head = (int)P.n_head, rb.n_kv_head = (int)P.n_kv_head, rb.neox = P.rope_neox;
            if (P.kv_f16) {
                if (hd == 64) {
                    rope_kv_batch_kernel<64, __half><<<(unsigned)n, 256, 0, stream>>>(rb);
                    attn_prefill_kernel<64, __half><<<ag, 256, 0, stream>>>(bqk, (const __half *)kc, (const __half *)vc, bxn, (int)n, (int)c0, (int)qd, (int)kvd, kvmul, scale);
                } else {
                    rope_kv_batch_kernel<128, __half><<<(unsigned)n, 256, 0, stream>>>(rb);
                    attn_prefill_kernel<128, __half><<<ag, 256, 0, stream>>>(bqk, (const __half *)kc, (const __half *)vc, bxn, (int)n, (int)c0, (int)qd, (int)kvd, kvmul, scale);
                }
            } else {
                if (hd == 64) {
                    rope_kv_batch_kernel<64, float><<<(unsigned)n, 256, 0, stream>>>(rb);
                    attn_prefill_kernel<64, float><<<ag, 256, 0, stream>>>(bqk, (const float *)kc, (const float *)vc, bxn, (int)n, (int)c0, (int)qd, (int)kvd, kvmul, scale);
                } else {
                    rope_kv_batch_kernel<128, float><<<(unsigned)n, 256, 0, stream>>>(rb);
                    attn_prefill_kernel<128, float><<<ag, 256, 0, stream>>>(bqk, (const float *)kc, (const float *)vc, bxn, (int)n, (int)c0, (int)qd, (int)kvd, kvmul, scale);
                }
            }
            TRY(cudaGetLastError());
            // the attention output [n, qd] sits in bxn; residual adds and silu(g)*u happen in the GEMM epilogues
            TRY(gemm(L.wo, bxn, bx, n, EPI_RESIDUAL, bx));
            rmsnorm_batch_kernel<<<(unsigned)n, 256, 0, stream>>>(bx, L.ffn_norm, P.eps, (int)E, bxn);
            TRY(gemm(L.wgu, bxn, bh, n, EPI_SWIGLU));
            TRY(gemm(L.wd, bh, bx, n, EPI_RESIDUAL, bx));
            TRY(cudaGetLastError());
        }
        if (c0 + n == s) { // the last token's hidden state -> final norm + output projection
            TRY(cudaMemcpyAsync(x, bx + (n - 1) * E, E * 4, cudaMemcpyDeviceToDevice, stream));
            TRY(mv(output, x, logits, final_norm, EPI_STORE, nullptr));
        }
    }
    TRY(cudaMemcpyAsync(h_logits, logits, P.vocab * 4, cudaMemcpyDeviceToHost, stream)); // page-locked staging, as in forward()
    TRY(cudaStreamSynchronize(stream));
#undef TRY
    memcpy(logits_host, h_logits, P.vocab * 4);
    return cudaSuccess;
}

// ---------------------------------------------------------------------------------------------------------------
// A tree of drafted tokens through every layer in one pass, against the cache (verify) and what is kept of it (accept)
// ---------------------------------------------------------------------------------------------------------------
// The engine's cache is the paged operators' pool with one page of n_ctx slots.
ullm_kv_pages Forward::pages() const {
    const size_t kvd = P.n_kv_head * P.head_dim;
    ullm_kv_pages kv;
    kv.dtype = P.kv_f16 ? ULLM_DTYPE_F16 : ULLM_DTYPE_F32, kv.n_layer = P.n_layer, kv.n_pages = 1, kv.page_size = P.n_ctx;
    kv.n_kv_head = P.n_kv_head, kv.head_dim = P.head_dim, kv.d_k = kcache, kv.d_v = vcache;
    kv.layer_stride = kv.page_stride = P.n_ctx * kvd, kv.slot_stride = kvd, kv.head_stride = P.head_dim;
    return kv;
}

// Device and page-locked int32 arrays of a tree step: table {block 0, length, count, fault, row 0, drafts, kept}, rows' offsets, parents,
// path, and per row sequence, slot, position and the bits of its ancestors.
namespace {
constexpr size_t VN = Forward::MAX_VERIFY, VW = VN / 32;
enum : size_t { V_BLOCK = 0, V_LEN = 1, V_REFS = 2, V_FAULT = 3, V_ROW = 4, V_DRAFT = 5, V_KEPT = 6, V_CU = 8, V_PARENT = 16, V_PATH = V_PARENT + VN, V_IN = V_PATH + VN,
               V_SEQ = V_IN, V_SLOT = V_SEQ + VN, V_POS = V_SLOT + VN, V_MASK = V_POS + VN, V_INTS = V_MASK + VN * VW };
}

cudaError_t Forward::verify_buffers(ullm_cuda_ctx *c) {
    cudaError_t e;
#define TRY(x) \
    if ((e = (x)) != cudaSuccess) return e;
    if (vready) return cudaSuccess;
    const size_t qd = P.n_head * P.head_dim, kvd = P.n_kv_head * P.head_dim;
    const ullm_kv_pages kv = pages();
    vwork_bytes = ullm_cuda_tree_attn_work_bytes(c, &kv, ULLM_DTYPE_F32), vtable_bytes = ullm_cuda_kv_work_bytes(1, 1);
    if (!vx) TRY(dev_alloc((void **)&vx, VN * P.n_embd * 4));
    if (!vxn) TRY(dev_alloc((void **)&vxn, VN * P.n_embd * 4));
    if (!vqkv) TRY(dev_alloc((void **)&vqkv, VN * (qd + 2 * kvd) * 4));
    if (!vattn) TRY(dev_alloc((void **)&vattn, VN * qd * 4));
    if (!vlogits) TRY(dev_alloc((void **)&vlogits, VN * P.vocab * 4));
    if (P.n_experts && !vrouter) TRY(dev_alloc((void **)&vrouter, VN * P.n_experts * 4));
    if (!vints) TRY(dev_alloc((void **)&vints, V_INTS * 4));
    if (!vwork) TRY(dev_alloc(&vwork, vwork_bytes));
    if (!vtable) TRY(dev_alloc(&vtable, vtable_bytes));
    if (!h_vints) TRY(cudaHostAlloc((void **)&h_vints, V_IN * 4, cudaHostAllocDefault));
    if (!h_vx) TRY(cudaHostAlloc((void **)&h_vx, VN * std::max(P.n_embd, P.vocab) * 4, cudaHostAllocDefault));
    if (batch_supported()) {
        TRY(batch_buffers());
        if (gemm_tc_supported(output.fmt, output.out, output.cols, 1)) {
            size_t bytes = 0;
            for (size_t n = 1; n <= VN; ++n) bytes = std::max(bytes, gemm_tc_scratch_bytes(output.out, output.cols, n, dev.sm_count));
            if (!vscratch) TRY(dev_alloc(&vscratch, bytes));
        }
    }
    vready = true;
#undef TRY
    return cudaSuccess;
}

int Forward::verify(ullm_cuda_ctx *c, const float *embeds, const int32_t *parents, size_t n, size_t pos, float *logits_host) {
    auto fail = [&](cudaError_t err) {
        cudaStreamSynchronize(stream); // (what was enqueued still reads the staging arrays)
        cudaGetLastError();
        if (err == cudaErrorNotSupported) return ctx_fail(c, ULLM_ERR_UNSUPPORTED, "a layer shape is outside the fused decode path");
        return ctx_fail(c, err == cudaErrorMemoryAllocation ? ULLM_ERR_OOM : ULLM_ERR_CUDA, "verifying a tree: %s", cudaGetErrorString(err));
    };
    auto drop = [&](int status) {
        cudaStreamSynchronize(stream);
        return status;
    };
    cudaError_t e;
    int rc;
#define TRY(x) \
    if ((e = (x)) != cudaSuccess) return fail(e);
    TRY(cudaSetDevice(device));
    TRY(verify_buffers(c));
    const size_t hd = P.head_dim, qd = P.n_head * hd, kvd = P.n_kv_head * hd, E = P.n_embd;
    const bool gemms = n >= VERIFY_GEMM_MIN && batch_supported();
    memset(h_vints, 0, V_PARENT * 4);
    h_vints[V_LEN] = (int)(pos + n), h_vints[V_CU + 1] = (int)n;
    for (size_t i = 0; i < n; ++i) h_vints[V_PARENT + i] = parents ? parents[i] : (int)i - 1;
    memcpy(h_vx, embeds, n * E * 4);
    TRY(cudaMemcpyAsync(vints, h_vints, V_PATH * 4, cudaMemcpyHostToDevice, stream));
    float *const xs = gemms ? bx : vx;
    TRY(cudaMemcpyAsync(xs, h_vx, n * E * 4, cudaMemcpyHostToDevice, stream));
    if ((rc = ullm_cuda_tree_plan_dev(c, n, 1, vints + V_CU, vints + V_LEN, nullptr, 1, vints + V_PARENT, vints + V_SEQ, vints + V_SLOT, vints + V_POS,
                                      (uint32_t *)vints + V_MASK, VW, vints + V_FAULT, stream)))
        return drop(rc);
    const ullm_kv_pages kv = pages();
    ullm_qk_norm_rope ro;
    memset(&ro, 0, sizeof ro);
    ro.kv = &kv, ro.x_dtype = ro.q_dtype = ULLM_DTYPE_F32, ro.n_rows = n, ro.n_head = P.n_head, ro.eps = P.eps, ro.d_rope = (const float *)rope, ro.n_pos = P.n_ctx;
    ro.neox = P.rope_neox, ro.d_row_seq = vints + V_SEQ, ro.d_row_slot = vints + V_SLOT, ro.d_row_pos = vints + V_POS, ro.d_blocks = vints + V_BLOCK;
    ro.n_table = ro.max_blocks = 1, ro.d_fault = vints + V_FAULT;
    ullm_tree_attn at;
    memset(&at, 0, sizeof at);
    at.kv = &kv, at.dtype = ULLM_DTYPE_F32, at.n_rows = n, at.n_seq = 1, at.n_head = P.n_head, at.d_cu = vints + V_CU, at.d_len = vints + V_LEN, at.d_blocks = vints + V_BLOCK;
    at.n_table = at.max_blocks = 1, at.d_mask = (const uint32_t *)vints + V_MASK, at.mask_words = VW, at.d_work = vwork, at.work_bytes = vwork_bytes;
    auto gemm = [&](const Mat &m, const float *in, float *out, int epi = EPI_STORE, const float *res = nullptr, void *scratch = nullptr) {
        return launch_gemm_tc(m.fmt, m.w, in, out, scratch ? scratch : bscratch, m.out, m.cols, n, dev.sm_count, d_status, stream, epi, res);
    };
    for (size_t l = 0; l < P.n_layer; ++l) {
        Layer &L = layers[l];
        float *qkv = vqkv, *attn_out = vattn;
        size_t ld = qd + 2 * kvd; // row of a token's projections
        const float *vsrc = vqkv + qd + kvd;
        size_t vld = ld;
        if (gemms) {
            rmsnorm_batch_kernel<<<(unsigned)n, 256, 0, stream>>>(bx, L.attn_norm, P.eps, (int)E, bxn);
            TRY(gemm(L.wqk, bxn, bqk));
            TRY(gemm(L.wv, bxn, bv));
            qkv = bqk, ld = qd + kvd, vsrc = bv, vld = kvd, attn_out = bxn;
        } else {
            for (size_t t = 0; t < n; ++t) {
                const float *x0 = vx + t * E;
                float *q0 = vqkv + t * ld;
                if (L.qkv_fused) {
                    TRY(mv(L.wqk, x0, q0, L.attn_norm, EPI_STORE, nullptr));
                    continue;
                }
                if (L.qk_fused) {
                    TRY(mv(L.wqk, x0, q0, L.attn_norm, EPI_STORE, nullptr));
                } else {
                    TRY(mv(L.wq, x0, q0, L.attn_norm, EPI_STORE, nullptr));
                    TRY(mv(L.wk, x0, q0 + qd, L.attn_norm, EPI_STORE, nullptr));
                }
                TRY(mv(L.wv, x0, q0 + qd + kvd, L.attn_norm, EPI_STORE, nullptr));
            }
        }
        ro.layer = at.layer = l;
        ro.d_q = ro.d_q_out = qkv, ro.d_k = qkv + qd, ro.d_v = vsrc, ro.q_stride = ro.k_stride = ro.q_out_stride = ld, ro.v_stride = vld;
        ro.d_q_norm = L.q_norm, ro.d_k_norm = L.k_norm, ro.d_q_bias = L.q_bias, ro.d_k_bias = L.k_bias, ro.d_v_bias = L.v_bias;
        if ((rc = ullm_cuda_qk_norm_rope_dev(c, &ro, stream))) return drop(rc);
        at.d_q = qkv, at.q_stride = ld, at.d_out = attn_out;
        if ((rc = ullm_cuda_tree_attn_dev(c, &at, stream))) return drop(rc);
        if (gemms) {
            TRY(gemm(L.wo, bxn, bx, EPI_RESIDUAL, bx));
            rmsnorm_batch_kernel<<<(unsigned)n, 256, 0, stream>>>(bx, L.ffn_norm, P.eps, (int)E, bxn);
            TRY(gemm(L.wgu, bxn, bh, EPI_SWIGLU));
            TRY(gemm(L.wd, bh, bx, EPI_RESIDUAL, bx));
            TRY(cudaGetLastError());
            continue;
        }
        for (size_t t = 0; t < n; ++t) {
            float *x0 = vx + t * E;
            TRY(mv(L.wo, vattn + t * qd, x0, nullptr, EPI_RESIDUAL, x0));
            if (L.moe) {
                TRY(mv(L.moe_gate, x0, vrouter + t * P.n_experts, L.ffn_norm, EPI_STORE, nullptr));
                continue;
            }
            if (!L.gu_fused) return fail(cudaErrorNotSupported);
            TRY(mv(L.wgu, x0, hidden, L.ffn_norm, EPI_SWIGLU, nullptr));
            TRY(mv(L.wd, hidden, x0, nullptr, EPI_RESIDUAL, x0));
        }
        if (L.moe) { // every expert that any of the tokens chose is read once
            // (eight tokens at a time: what one call takes in one go, so that a refusal has changed nothing yet)
            for (size_t t = 0; t < n; t += 8) {
                const size_t nt = std::min((size_t)8, n - t);
                float *x0 = vx + t * E;
                const float *r0 = vrouter + t * P.n_experts;
                e = launch_moe_ffn(dev, L.experts, x0, r0, nt, P.n_experts_used, x0, nullptr, nullptr, moe_scratch, d_status, stream, false, use_pdl, nullptr, x0, L.ffn_norm,
                                   P.eps);
                if (e == cudaErrorNotSupported) { // shapes outside the streamed kernels go through a normalised copy, as in the decode step
                    cudaGetLastError();
                    rmsnorm_batch_kernel<<<(unsigned)nt, 256, 0, stream>>>(x0, L.ffn_norm, P.eps, (int)E, vxn);
                    TRY(cudaGetLastError());
                    e = launch_moe_ffn(dev, L.experts, vxn, r0, nt, P.n_experts_used, x0, nullptr, nullptr, moe_scratch, d_status, stream, false, use_pdl, nullptr, x0);
                }
                TRY(e);
            }
        }
    }
    if (gemms && vscratch) {
        rmsnorm_batch_kernel<<<(unsigned)n, 256, 0, stream>>>(bx, final_norm, P.eps, (int)E, bxn);
        TRY(gemm(output, bxn, vlogits, EPI_STORE, nullptr, vscratch));
    } else {
        for (size_t t = 0; t < n; ++t) TRY(mv(output, xs + t * E, vlogits + t * P.vocab, final_norm, EPI_STORE, nullptr));
    }
    TRY(cudaMemcpyAsync(h_vx, vlogits, n * P.vocab * 4, cudaMemcpyDeviceToHost, stream)); // page-locked staging, as in forward()
    TRY(cudaStreamSynchronize(stream));
    memcpy(logits_host, h_vx, n * P.vocab * 4);
    return ctx_check_status(c); // (the tree operators' waits report to the context)
}

int Forward::accept(ullm_cuda_ctx *c, size_t pos, size_t n, const int32_t *path, size_t kept) {
    cudaError_t e;
    DeviceGuard guard(c->device);
    if ((e = verify_buffers(c)) != cudaSuccess) {
        cudaGetLastError();
        return ctx_fail(c, e == cudaErrorMemoryAllocation ? ULLM_ERR_OOM : ULLM_ERR_CUDA, "accept: %s", cudaGetErrorString(e));
    }
    memset(h_vints, 0, V_PARENT * 4);
    h_vints[V_LEN] = (int)(pos + n), h_vints[V_REFS] = 1, h_vints[V_DRAFT] = (int)n, h_vints[V_KEPT] = (int)kept;
    for (size_t j = 0; j < kept; ++j) h_vints[V_PATH + j] = path[j];
    const ullm_kv_pages kv = pages();
    ullm_kv_table t;
    t.d_blocks = vints + V_BLOCK, t.d_len = vints + V_LEN, t.d_refs = vints + V_REFS, t.d_fault = vints + V_FAULT, t.n_seq = 1, t.max_blocks = 1;
    t.d_work = vtable, t.work_bytes = vtable_bytes;
    ULLM_CUDA_TRY(c, cudaMemcpyAsync(vints, h_vints, V_IN * 4, cudaMemcpyHostToDevice, stream));
    int rc = ullm_cuda_kv_accept_dev(c, &kv, &t, vints + V_ROW, vints + V_DRAFT, vints + V_PATH, vints + V_KEPT, 1, VN, stream);
    const cudaError_t done = cudaStreamSynchronize(stream); // (the staging array is free again)
    if (rc) return rc;
    ULLM_CUDA_TRY(c, done);
    return ULLM_OK;
}
#undef TRY

} // namespace ullm
