// How the attention over a paged cache is divided among CTAs.
//
// A unit of work is (sequence, key head, tile of M query rows); a query row is (row of the step, query head of the
// group), so that a group's heads share every key that is loaded.  A unit takes its key blocks in order.  All units'
// blocks are laid end to end and every CTA takes an equal contiguous part of that line, whatever the
// lengths are: one long sequence fills the machine as well as a thousand short ones.  A unit that is cut leaves unnormalised
// partial results (running maximum, sum and weighted values of each row) in the work area; a CTA has at most two of
// them, its first and its last, and the CTA in which a cut unit ends records what the joining kernel needs.
// Lengths are read on the device, so a captured call serves every later state of the tables.
#pragma once

#include "paged.h"

namespace ullm {

struct SeqView {
    int r0, n;   // its rows
    int id;      // its table row
    int ctx, kv; // tokens in front of the rows; keys in all (0: nothing to see, rows become zeros)
};
__device__ __forceinline__ SeqView seq_view(const TreeDev &p, int b) {
    SeqView v;
    v.r0 = p.cu[b];
    const int r1 = p.cu[b + 1];
    v.id = p.ids ? p.ids[b] : b;
    v.n = v.r0 < 0 || r1 < v.r0 || r1 > p.n_rows ? 0 : r1 - v.r0;
    const bool known = v.id >= 0 && v.id < p.n_table;
    const int len = known ? p.len[v.id] : -1;
    if (len < v.n || len > (long long)p.max_blocks * p.page_size) v.ctx = v.kv = 0;
    else v.ctx = len - v.n, v.kv = len;
    if (!known) v.id = 0;
    return v;
}
// Whether row `i` of a sequence sees node `j` of the sequence's rows (0 <= j < n).
__device__ __forceinline__ bool sees(const TreeDev &p, const SeqView &v, int i, int j) {
    if (!p.mask) return j <= i;
    if (j >= 32 * p.mask_words) return false;
    return (p.mask[(size_t)(v.r0 + i) * p.mask_words + (j >> 5)] >> (j & 31)) & 1u;
}

template <int M, int KB> struct Tiles {
    static __device__ __forceinline__ int count(const TreeDev &p, const SeqView &v) { return (v.n * p.group + M - 1) / M; }
    // one behind the last key that a tile's rows can see
    static __device__ __forceinline__ int key_end(const TreeDev &p, const SeqView &v, int t) {
        if (p.mask || !v.kv) return v.kv;
        return v.ctx + min((int)(((t + 1u) * M - 1u) / (unsigned)p.group), v.n - 1) + 1;
    }
    static __device__ __forceinline__ int blocks(const TreeDev &p, const SeqView &v, int t) { return max(1, (key_end(p, v, t) + KB - 1) / KB); }
    // blocks of all tiles of one key head
    static __device__ __forceinline__ long long per_head(const TreeDev &p, const SeqView &v) {
        const int T = count(p, v);
        if (!T) return 0;
        if (p.mask || T == 1) return (long long)T * blocks(p, v, 0);
        long long s = 0;
        for (int t = 0; t < T; ++t) s += blocks(p, v, t);
        return s;
    }
};

struct Share { // of one CTA
    long long total, lo, hi;
    int active; // CTAs that have a share
    int b;      // sequence in which it begins
    long long base; // blocks in front of that sequence
};
__device__ __forceinline__ long long share_at(long long total, int active, long long c) { return total * c / active; }

// Sum over the CTA and exclusive prefix, NT threads (a multiple of 32).
template <int NT> __device__ __forceinline__ long long cta_scan64(long long v, long long *excl, long long *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        const long long s = warp_sums[w];
        if (w < warp) before += s;
        all += s;
    }
    *excl = before + x - v;
    return all;
}

// Every thread of the CTA calls it; MINB: a CTA takes at least so many blocks where there are few.
template <int M, int KB, int NT, int MINB> __device__ __forceinline__ Share cta_share(const TreeDev &p) {
    __shared__ long long sums[NT / 32];
    __shared__ long long s_base;
    __shared__ int s_b;
    Share s;
    s.total = 0;
    long long work = 0, excl = 0;
    for (int b0 = 0; b0 < p.n_seq; b0 += NT) {
        const int b = b0 + threadIdx.x;
        work = b < p.n_seq ? Tiles<M, KB>::per_head(p, seq_view(p, b)) * p.n_kv : 0;
        s.total += cta_scan64<NT>(work, &excl, sums);
    }
    const long long wanted = (s.total + MINB - 1) / MINB;
    s.active = (int)max(1ll, min((long long)gridDim.x, wanted));
    s.b = 0, s.base = 0, s.lo = s.hi = 0;
    if ((int)blockIdx.x >= s.active || s.total == 0) return s;
    s.lo = share_at(s.total, s.active, blockIdx.x), s.hi = share_at(s.total, s.active, blockIdx.x + 1);
    long long run = 0;
    for (int b0 = 0; b0 < p.n_seq; b0 += NT) {
        const int b = b0 + threadIdx.x;
        long long sum;
        if (p.n_seq > NT) {
            work = b < p.n_seq ? Tiles<M, KB>::per_head(p, seq_view(p, b)) * p.n_kv : 0;
            sum = cta_scan64<NT>(work, &excl, sums);
        } else {
            sum = s.total;
        }
        if (s.lo >= run + excl && s.lo < run + excl + work) s_b = b, s_base = run + excl;
        run += sum;
        if (run > s.lo) break;
    }
    __syncthreads();
    s.b = s_b, s.base = s_base;
    return s;
}

// Steps through a CTA's share, one segment (the part of one unit that lies in it) at a time.
template <int M, int KB> struct Walk {
    using T = Tiles<M, KB>;
    const TreeDev &p;
    const Share &s;
    long long cur;
    SeqView v;
    int b, h, t, nt, blk; // the segment: key head, tile, first block ...
    int nb, end;          // ... blocks of its unit, one behind its last block
    __device__ Walk(const TreeDev &p_, const Share &s_) : p(p_), s(s_), cur(s_.lo), b(s_.b) {
        if (cur >= s.hi) return;
        v = seq_view(p, b);
        nt = T::count(p, v);
        const long long per = T::per_head(p, v);
        long long o = cur - s.base;
        h = (int)(o / per);
        o -= h * per;
        t = 0;
        if (p.mask) {
            nb = T::blocks(p, v, 0);
            t = (int)(o / nb), blk = (int)(o % nb);
        } else {
            for (nb = T::blocks(p, v, 0); o >= nb; nb = T::blocks(p, v, ++t)) o -= nb;
            blk = (int)o;
        }
        end = blk + (int)min((long long)(nb - blk), s.hi - cur);
    }
    __device__ bool more() const { return cur < s.hi; }
    __device__ bool first() const { return cur == s.lo; }
    __device__ bool whole() const { return blk == 0 && end == nb; }
    // where a cut unit's partial result goes
    __device__ int slot() const { return first() ? 0 : 1; }
    __device__ void next() {
        cur += end - blk;
        if (cur >= s.hi) return;
        blk = 0;
        if (++t == nt) {
            t = 0;
            if (++h == p.n_kv) {
                h = 0;
                do {
                    v = seq_view(p, ++b);
                    nt = T::count(p, v);
                } while (nt == 0);
            }
        }
        nb = T::blocks(p, v, t);
        end = (int)min((long long)nb, s.hi - cur);
    }
    // What the joining kernel needs of the CTA in which a cut unit ends: the CTA and slot in which it begins.
    __device__ void record(int4 *meta) const {
        if (blk == 0 || end != nb) return;
        const long long start = cur - blk;
        long long c0 = start * s.active / s.total;
        while (share_at(s.total, s.active, c0 + 1) <= start) ++c0;
        while (share_at(s.total, s.active, c0) > start) --c0;
        meta[0] = make_int4((int)c0, share_at(s.total, s.active, c0) == start ? 0 : 1, v.r0, v.n);
        meta[1] = make_int4(t, h, 0, 0);
    }
};

// Partial results of slot 0 / 1 of CTA c: M rows of dim values, then M pairs (maximum, sum).
template <int M> __device__ __forceinline__ float *part_of(const TreeDev &p, int c, int slot) {
    return p.part + ((size_t)c * 2 + slot) * M * (p.dim + 2);
}

template <typename T> __device__ __forceinline__ T out_from(float v);
template <> __device__ __forceinline__ float out_from<float>(float v) { return v; }
template <> __device__ __forceinline__ __half out_from<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 out_from<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Joins the parts of the unit that ends in CTA blockIdx.x, in the order of the CTAs: a row per warp.
// out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c.
template <typename O, int M> __global__ void __launch_bounds__(256) tree_join_kernel(const TreeDev p) {
    pdl_wait_prior();
    pdl_launch_dependents();
    const int c = blockIdx.x, lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
    const int4 a = p.meta[c * TREE_META], b = p.meta[c * TREE_META + 1];
    if (a.x < 0) return;
    const long long row = (long long)b.x * M + r;
    if (row >= (long long)a.w * p.group) return;
    const int parts = c - a.x + 1;
    auto part = [&](int k) { return part_of<M>(p, a.x + k, k == 0 ? a.y : 0); };
    float m = -INFINITY;
    for (int k = lane; k < parts; k += 32) m = fmaxf(m, part(k)[(size_t)M * p.dim + 2 * r]);
    m = warp_max(m);
    float l = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
        float w = 0.f;
        if (k0 + lane < parts) {
            const float2 ml = *(const float2 *)(part(k0 + lane) + (size_t)M * p.dim + 2 * r);
            w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
            l += ml.y * w;
        }
        for (int k = 0; k < min(32, parts - k0); ++k) {
            const float wk = __shfl_sync(0xffffffffu, w, k);
            if (wk == 0.f) continue; // an empty part's values were never written
            const float *o = part(k0 + k) + (size_t)r * p.dim;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (lane + 32 * e < p.dim) acc[e] += wk * o[lane + 32 * e];
        }
    }
    l = warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    O *out = (O *)p.out + (a.z + row / p.group) * p.out_stride + ((long long)b.y * p.group + row % p.group) * p.dim;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < p.dim) out[lane + 32 * e] = out_from<O>(l == 0.f ? 0.f : acc[e] * inv);
}

} // namespace ullm
