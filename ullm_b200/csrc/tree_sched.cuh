// How the attention over a paged cache is divided among CTAs.
//
// A unit of work is (sequence, key head, tile of M query rows); a query row is (row of the step, query head of the
// group), so that a group's heads share every key that is loaded.  A unit takes its key blocks in order.  All units'
// blocks are laid end to end, each unit led in by COST places for what it costs to begin and to end one, and every CTA
// takes an equal contiguous part of that line, whatever the lengths are: one long sequence fills the machine as well as a
// thousand short ones.  A unit that is cut leaves unnormalised partial results (running maximum, sum and
// weighted values of each row) in the work area; a CTA has at most two of them, its first and its last, and the CTA in
// which a cut unit ends records what the joining kernel needs.  Lengths are read on the device, so a captured call serves
// every later state of the tables.  Where sequences have many rows, `lanes` CTAs form a team that shares one line: its
// members take neighbouring tiles of a unit over the same keys at about the same time, so that the keys come from DRAM once and
// from the L2 afterwards (each tile at a time of its own: 437 MB of keys and values were read four times).  One warp of a CTA works the division out (Sched) and hands the segments to the others:
// done by every thread, with 64-bit divisions, it took 6,000 of the 13,800 cycles of a one-token call.
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
};

// The part of one unit that lies in a CTA's share.
struct __align__(16) Seg {
    int r0, n, id, ctx, kv;       // the sequence (SeqView)
    int key_end;                  // one behind the last key that the tile's rows see
    int h, row0, rows;            // key head; first row of the tile among the sequence's query rows, and how many there are
    int blk, count;               // first key block, blocks (0: no more segments)
    int flags;                    // 1: the whole unit; 2: its partial result goes to slot 1
    short odd, big;               // set by who finds values that are not finite, or queries beyond what a kernel's quick way takes
    int first, parts, end;        // of a unit that was cut: the CTA that begins it (<< 1 | its slot there), the CTAs that have a part of it, the one that ends it
};

template <int M, int KB, int COST, int MINS> struct Sched {
    using T = Tiles<M, KB>;
    static constexpr unsigned ALL = 0xffffffffu;
    const TreeDev &p;
    const int lane;
    const int shift, lanes, member, team; // CTAs of a team (a power of two), this one's place in it, the team
    unsigned total, active, each, more, lo, hi, cur; // share c begins at c * each + min(c, more)
    int b, h, t, nt;
    unsigned off; // place of `cur` in its unit
    SeqView win;  // view of sequence wb + lane
    int wb;
    SeqView v;

    __device__ __forceinline__ explicit Sched(const TreeDev &p_, int shift_ = 0)
        : p(p_), lane((int)(threadIdx.x & 31)), shift(shift_), lanes(1 << shift_), member((int)blockIdx.x & ((1 << shift_) - 1)), team((int)blockIdx.x >> shift_) {}
    // tiles that a team takes together, and their places: those of the one that sees most
    __device__ __forceinline__ int groups(const SeqView &u) const { return (T::count(p, u) + lanes - 1) >> shift; }
    __device__ __forceinline__ int group_blocks(const SeqView &u, int g) const { return T::blocks(p, u, min((g + 1) * lanes, T::count(p, u)) - 1); }

    __device__ __forceinline__ unsigned share_at(unsigned c) const { return c * each + min(c, more); }
    __device__ __forceinline__ unsigned share_of(unsigned x) const { // the share that holds place x
        const unsigned big = more * (each + 1);
        return x < big ? x / (each + 1) : more + (x - big) / each;
    }
    // places of one key head of the sequence that lane `who` views (`mine`: this lane's); every lane calls it
    __device__ __forceinline__ unsigned head_places(const SeqView &mine) const {
        const int T_ = groups(mine);
        const bool simple = p.mask || T_ <= 8;
        unsigned s = 0;
        if (p.mask) {
            s = T_ ? (unsigned)T_ * (T::blocks(p, mine, 0) + COST) : 0u;
        } else if (simple) {
            for (int i = 0; i < T_; ++i) s += group_blocks(mine, i) + COST;
        }
        for (unsigned long_ones = __ballot_sync(ALL, !simple); long_ones; long_ones &= long_ones - 1) { // prompts: all lanes together
            const int who = __ffs(long_ones) - 1;
            const SeqView u = view_of(mine, who);
            const int n = groups(u);
            unsigned x = 0;
            for (int i = lane; i < n; i += 32) x += group_blocks(u, i) + COST;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
            if (lane == who) s = x;
        }
        return s;
    }
    __device__ __forceinline__ SeqView view_of(const SeqView &mine, int who) const {
        SeqView u;
        u.r0 = __shfl_sync(ALL, mine.r0, who), u.n = __shfl_sync(ALL, mine.n, who), u.id = __shfl_sync(ALL, mine.id, who);
        u.ctx = __shfl_sync(ALL, mine.ctx, who), u.kv = __shfl_sync(ALL, mine.kv, who);
        return u;
    }
    __device__ __forceinline__ SeqView lane_view(int b0) const {
        SeqView u;
        u.r0 = u.n = u.id = u.ctx = u.kv = 0;
        if (b0 + lane < p.n_seq) u = seq_view(p, b0 + lane);
        return u;
    }
    // Works out the CTA's share; false: it has none.
    __device__ __forceinline__ bool init() {
        total = 0;
        unsigned places = 0;
        for (int b0 = 0; b0 < p.n_seq; b0 += 32) {
            win = lane_view(b0), wb = b0;
            places = head_places(win) * (unsigned)p.n_kv;
            unsigned x = places;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
            total += x;
        }
        active = max(1u, min(gridDim.x >> shift, (total + MINS - 1) / MINS));
        each = total / active, more = total - each * active;
        if ((unsigned)team >= active || total == 0) return false;
        lo = share_at(team), hi = share_at(team + 1), cur = lo;
        unsigned run = 0; // places in front of the window
        for (int b0 = 0; b0 < p.n_seq; b0 += 32) {
            if (p.n_seq > 32) win = lane_view(b0), wb = b0, places = head_places(win) * (unsigned)p.n_kv;
            unsigned incl = places;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(ALL, incl, o);
                if (lane >= o) incl += y;
            }
            const unsigned here = __ballot_sync(ALL, lo < run + incl && lo >= run + incl - places);
            if (here) {
                const int who = __ffs(here) - 1;
                off = lo - (run + __shfl_sync(ALL, incl - places, who));
                b = b0 + who;
                break;
            }
            run += __shfl_sync(ALL, incl, 31);
        }
        v = view_of(win, b - wb), nt = groups(v);
        const unsigned per = __shfl_sync(ALL, places / (unsigned)p.n_kv, b - wb);
        h = (int)(off / per), off -= h * per, t = 0;
        if (p.mask) {
            const unsigned u = T::blocks(p, v, 0) + COST;
            t = (int)(off / u), off -= t * u;
        } else {
            for (int t0 = 0;; t0 += 32) { // the tile, 32 at a time
                const unsigned mine = t0 + lane < nt ? group_blocks(v, t0 + lane) + COST : 0u;
                unsigned incl = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned y = __shfl_up_sync(ALL, incl, o);
                    if (lane >= o) incl += y;
                }
                const unsigned here = __ballot_sync(ALL, off < incl && off >= incl - mine);
                if (here) {
                    t = t0 + __ffs(here) - 1, off -= __shfl_sync(ALL, incl - mine, t - t0);
                    break;
                }
                off -= __shfl_sync(ALL, incl, 31);
            }
        }
        return true;
    }
    // The next segment; count 0 when the share is used up.  meta: where the joining kernel's record goes; null: the segment says who joins (join_last).
    __device__ __forceinline__ Seg next(int4 *meta) {
        Seg s;
        s.count = 0, s.odd = s.big = 0;
        while (cur < hi) {
            const int nb = group_blocks(v, t), tile = t * lanes + member;
            const unsigned len = nb + COST, take = min(len - off, hi - cur);
            // this member's tile: it may be missing, or see fewer keys than the group's last
            const int mine = tile * M < v.n * p.group ? T::blocks(p, v, tile) : 0;
            const int b0 = max((int)off - COST, 0), b1 = min((int)(off + take) - COST, mine);
            if (b1 > b0) {
                s.r0 = v.r0, s.n = v.n, s.id = v.id, s.ctx = v.ctx, s.kv = v.kv, s.key_end = T::key_end(p, v, tile);
                s.h = h, s.row0 = tile * M, s.rows = min(M, v.n * p.group - tile * M);
                s.blk = b0, s.count = b1 - b0;
                const bool whole = b0 == 0 && b1 == mine;
                s.flags = (whole ? 1 : 0) | (cur == lo ? 0 : 2); // slot 0: the unit with which the share begins
                if (!whole && !meta) {
                    const unsigned unit = cur - off, c0 = share_of(unit + COST), c1 = share_of(unit + COST + mine - 1); // the teams that hold its first and its last block
                    s.first = (int)(c0 * lanes + member) << 1 | (share_at(c0) >= unit ? 0 : 1), s.parts = (int)(c1 - c0) + 1, s.end = (int)c1 * lanes + member;
                } else if (!whole && b1 == mine && lane == 0) {
                    const unsigned unit = cur - off, c0 = share_of(unit + COST); // the team that holds its first block
                    meta[0] = make_int4((int)c0 * lanes + member, (share_at(c0) >= unit ? 0 : 1) | lanes << 1, v.r0, v.n);
                    meta[1] = make_int4(tile, h, 0, 0);
                }
            }
            cur += take, off = 0;
            if (cur < hi && ++t == nt) {
                t = 0;
                if (++h == p.n_kv) {
                    h = 0;
                    do {
                        if (++b - wb == 32) win = lane_view(b), wb = b;
                        v = view_of(win, b - wb), nt = groups(v);
                    } while (nt == 0);
                }
            }
            if (s.count) break;
        }
        return s;
    }
};

// Partial results of slot 0 / 1 of CTA c: M rows of dim values, then M pairs (maximum, sum).
template <int M> __device__ __forceinline__ float *part_of(const TreeDev &p, int c, int slot) {
    return p.part + ((size_t)c * 2 + slot) * M * (p.dim + 2);
}

// Four neighbouring values as f32
__device__ __forceinline__ float4 widen4(const float *p) { return *(const float4 *)p; }
__device__ __forceinline__ float4 widen4(const __half *p) {
    const uint2 v = *(const uint2 *)p;
    const float2 a = __half22float2(*(const __half2 *)&v.x), b = __half22float2(*(const __half2 *)&v.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 widen4(const __nv_bfloat16 *p) {
    const uint2 v = *(const uint2 *)p;
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
__device__ __forceinline__ void copy16(void *dst, const void *src, bool on) { // zeros where it is off
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// Values that are not finite, of keys that a row sees, decide what becomes of the row, however small their weights: products of a weight that has become
// zero in 32 bits or fewer with an infinity would be NaN where the formula has an infinity.  The kernels add up such values alone and put the sum in
// the place of what the products gave.  A key whose score is -inf does have no weight: an infinite value of it makes NaN, as in the formula.
template <typename Q, typename KV> __device__ __noinline__ bool has_no_weight(const Q *q, const KV *k, int dim, float scale) {
    float s = 0.f;
    for (int d = 0; d < dim; ++d) s = fmaf((float)q[d], (float)k[d], s);
    return s * scale == -INFINITY;
}

template <typename T> __device__ __forceinline__ T out_from(float v);
template <> __device__ __forceinline__ float out_from<float>(float v) { return v; }
template <> __device__ __forceinline__ __half out_from<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 out_from<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Weight of a part: 0 where nothing was seen, else at least the smallest number, so that an infinite value in it stays infinite.
__device__ __forceinline__ float part_weight(float m_part, float m) { return m_part == -INFINITY ? 0.f : fmaxf(exp2f(m_part - m), 1.4e-45f); }

// Joins a unit's parts in the kernel that made them: the CTAs that have a part of it count, and the last one to arrive joins them all, in the order of the CTAs.
// The counts are zeros when the kernel starts (tree_count_kernel).  Every thread calls it, behind its stores of the CTA's own part.
template <typename O, int M, int D> __device__ __forceinline__ void join_last(const TreeDev &p, const Seg &w, int *flag) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *flag = atomicAdd(p.count + w.end, 1) + 1 == w.parts;
    __syncthreads();
    if (!*flag) return;
    __threadfence();
    const int size = M * (D + 2), c0 = w.first >> 1;
    for (int i = threadIdx.x; i < w.rows * (D / 4); i += blockDim.x) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < w.parts; k0 += 8) { // eight parts on their way at once
            float4 x[8];
            float2 ml[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float *const part = p.part + ((c0 + k0 + k) * 2 + (k0 + k == 0 ? w.first & 1 : 0)) * size;
                ml[k] = make_float2(-INFINITY, 0.f), x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k0 + k < w.parts) ml[k] = __ldcg((const float2 *)(part + M * D + 2 * r)), x[k] = __ldcg((const float4 *)(part + r * D + d));
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
            const float corr = part_weight(m, top);
            if (m != -INFINITY) l *= corr, acc.x *= corr, acc.y *= corr, acc.z *= corr, acc.w *= corr;
            m = top;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float c = part_weight(ml[k].x, m);
                l += ml[k].y * c; // (NaN where a score was NaN)
                acc.x += c * x[k].x, acc.y += c * x[k].y, acc.z += c * x[k].z, acc.w += c * x[k].w;
            }
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const int row = w.row0 + r;
        O *const out = (O *)p.out + (w.r0 + row / p.group) * p.out_stride + ((long long)w.h * p.group + row % p.group) * D + d;
        const float y[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = out_from<O>(l == 0.f ? 0.f : y[e] * inv);
    }
}

// Joins the parts of the units that were cut, in the order of the CTAs:
//   out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c.
// A fixed number of CTAs share the rows of all cut units; every CTA reads the records.  The kernel is bound by round trips to memory: a row's values, references
// and sums are all on their way at once, since with weights first and values after them a row took 6,500 cycles.  Four warps take a row together (or one,
// where that saves passes), each every fourth part, up to eight at a time.  Behind tiles of 256 rows there are many more rows than warps, of two or three parts
// each: a warp then has eight parts of two or four rows on their way (join_rows; 12 sequences of 64 rows: 247 -> 230 us in all; it is no gain, and 1 to 3 us
// slower, where rows are few).
constexpr int JOIN_WARPS = 8, JOIN_MAX = 512; // JOIN_MAX: CTAs of the attention kernel at most
// CTAs on an SM, as many as are launched: registers for the loads on their way count for more than warps (general form: 2 for 12.2 us on a one-token call,
// 4 for 15.7)
template <int M> constexpr int JOIN_PER_SM = M >= 256 ? 3 : 2;
struct Duty {                 // a unit that was cut
    int front;                // rows of the units in front of it
    short c, c0;              // the CTAs in which it ends and begins ...
    int r0, t;
    unsigned short h, how;    // how: slot | lanes << 1
};
struct JoinShared {
    Duty duty[JOIN_MAX];
    int found[JOIN_WARPS], rows[JOIN_WARPS], most[JOIN_WARPS];
    float acc[JOIN_WARPS][256], l[JOIN_WARPS];
};

// K: parts of a row on their way at once, 8 / K rows per warp
template <typename O, int M, int K> __device__ __forceinline__ void join_rows(const TreeDev &p, JoinShared &sm, int n_duty, int n_rows) {
    constexpr int R = 8 / K, PER = JOIN_WARPS * R;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.dim;
    for (int first = blockIdx.x * PER; first < n_rows; first += gridDim.x * PER) {
        // lane L, L + 8, ... stand for part L % K of row L / K
        const int i = first + warp * R + (lane & 7) / K, k = lane % K;
        int parts = 0, at = 0, step = 0, at0 = 0, pair = 0, pair0 = 0; // places in floats: of part k * step behind at, of the first one at at0; and of the pairs
        long long out = 0;
        if (i < n_rows) {
            int lo = 0, hi = n_duty; // the unit of row i
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (sm.duty[mid].front <= i) lo = mid;
                else hi = mid;
            }
            const Duty u = sm.duty[lo];
            const int r = i - u.front, lanes = u.how >> 1, size = M * (D + 2), row = u.t * M + r;
            parts = (u.c - u.c0) / lanes + 1, step = lanes * 2 * size, at = u.c0 * 2 * size + r * D, at0 = at + (u.how & 1) * size;
            pair = u.c0 * 2 * size + M * D + 2 * r, pair0 = pair + (u.how & 1) * size;
            out = (u.r0 + row / p.group) * p.out_stride + ((long long)u.h * p.group + row % p.group) * D;
        }
        auto pair_of = [&](int j) { return j < parts ? *(const float2 *)(p.part + (j == 0 ? pair0 : pair + j * step)) : make_float2(-INFINITY, 0.f); };
        for (int d0 = 0; d0 < D; d0 += 128) {
            const int d = d0 + lane * 4;
            float m = -INFINITY, l = 0.f;
            float4 acc[R];
#pragma unroll
            for (int a = 0; a < R; ++a) acc[a] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j0 = 0; K < 8 ? j0 == 0 : j0 < parts; j0 += K) {
                const int j = j0 + k;
                const int mine = j < parts ? (j == 0 ? at0 : at + j * step) : -1;
                float4 x[8];
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const int from = __shfl_sync(0xffffffffu, mine, s);
                    x[s] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (from >= 0 && d < D) x[s] = *(const float4 *)(p.part + from + d);
                }
                const float2 ml = pair_of(j);
                if (j0 == 0) { // the row's reference, over all parts
                    if (K == 8) {
                        for (int q = lane; q < parts; q += 32) m = fmaxf(m, pair_of(q).x);
                        m = warp_max(m);
                    } else {
                        m = ml.x;
#pragma unroll
                        for (int o = K / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    }
                }
                const float w = part_weight(ml.x, m);
                l += ml.y * w;
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const float ws = __shfl_sync(0xffffffffu, w, s);
                    if (ws == 0.f) continue; // (an empty part's values were never written)
                    acc[s / K].x += ws * x[s].x, acc[s / K].y += ws * x[s].y, acc[s / K].z += ws * x[s].z, acc[s / K].w += ws * x[s].w;
                }
            }
#pragma unroll
            for (int o = K / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
            for (int a = 0; a < R; ++a) {
                const float la = __shfl_sync(0xffffffffu, l, a * K), inv = la == 0.f ? 0.f : 1.0f / la;
                const long long to = __shfl_sync(0xffffffffu, out, a * K);
                const bool there = __shfl_sync(0xffffffffu, parts, a * K) > 0;
                if (!there || d >= D) continue;
                O *const o = (O *)p.out + to + d;
                const float y[4] = {acc[a].x, acc[a].y, acc[a].z, acc[a].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = out_from<O>(la == 0.f ? 0.f : y[e] * inv);
            }
        }
    }
}

template <typename O, int M> __global__ void __launch_bounds__(32 * JOIN_WARPS, JOIN_PER_SM<M>) tree_join_kernel(const TreeDev p, int ctas) {
    __shared__ JoinShared sm;
    pdl_wait_prior();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = p.dim;
    int n_duty = 0, n_rows = 0, most = 0;
    for (int c0 = 0; c0 < ctas; c0 += 32 * JOIN_WARPS) {
        const int c = c0 + tid;
        int4 a = make_int4(-1, 0, 0, 0), b = a;
        if (c < ctas) a = p.meta[c * TREE_META], b = p.meta[c * TREE_META + 1];
        const bool has = a.x >= 0;
        const int r = has ? min(M, a.w * p.group - b.x * M) : 0;
        int incl = r, parts = has ? (c - a.x) / (a.y >> 1) + 1 : 0;
        const unsigned who = __ballot_sync(0xffffffffu, has);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
            parts = max(parts, __shfl_xor_sync(0xffffffffu, parts, o));
        }
        __syncthreads();
        if (lane == 31) sm.found[warp] = __popc(who), sm.rows[warp] = incl, sm.most[warp] = parts;
        __syncthreads();
        int at = n_duty + __popc(who & ((1u << lane) - 1u)), front = n_rows + incl - r;
        for (int k = 0; k < JOIN_WARPS; ++k) {
            if (k < warp) at += sm.found[k], front += sm.rows[k];
            n_duty += sm.found[k], n_rows += sm.rows[k], most = max(most, sm.most[k]);
        }
        if (has) {
            Duty d;
            d.front = front, d.c = (short)c, d.c0 = (short)a.x, d.r0 = a.z, d.t = b.x, d.h = (unsigned short)b.y, d.how = (unsigned short)a.y;
            sm.duty[at] = d;
        }
    }
    __syncthreads();
    if constexpr (M >= 256) {
        if (most <= 2) join_rows<O, M, 2>(p, sm, n_duty, n_rows);
        else if (most <= 4) join_rows<O, M, 4>(p, sm, n_duty, n_rows);
        else join_rows<O, M, 8>(p, sm, n_duty, n_rows);
        return;
    }
    // four warps to a row where that takes fewer round trips: passes over the rows times loads in turn per row
    const int warps = gridDim.x * JOIN_WARPS;
    const bool shared = (n_rows * 4 + warps - 1) / warps * ((most + 31) / 32) < (n_rows + warps - 1) / warps * ((most + 7) / 8);
    const int split = shared ? 4 : 1, per = JOIN_WARPS / split, sub = warp % split, wide = D <= 128 ? 4 : 8;
    const bool on = lane * wide < D;
    for (int i0 = blockIdx.x * per; i0 < n_rows; i0 += gridDim.x * per) {
        const int i = i0 + warp / split;
        float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        Duty u;
        int r = 0;
        if (i < n_rows) {
            int lo = 0, hi = n_duty; // the unit of row i
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (sm.duty[mid].front <= i) lo = mid;
                else hi = mid;
            }
            u = sm.duty[lo];
            r = i - u.front;
            const int lanes = u.how >> 1, parts = (u.c - u.c0) / lanes + 1;
            auto part = [&](int k) { return part_of<M>(p, u.c0 + k * lanes, k == 0 ? u.how & 1 : 0); };
            auto pair = [&](int k) { return k < parts ? *(const float2 *)(part(k) + (size_t)M * D + 2 * r) : make_float2(-INFINITY, 0.f); };
            for (int j0 = sub; j0 < parts; j0 += 8 * split) { // this warp's parts j0, j0 + split, ...
                const int n = min(8, (parts - j0 + split - 1) / split);
                float4 x[8];
                if (wide == 4) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < n && on) x[j] = *(const float4 *)(part(j0 + j * split) + (size_t)r * D + lane * 4);
                }
                if (j0 == sub) { // the row's reference, over all parts
                    for (int k = lane; k < parts; k += 32) m = fmaxf(m, pair(k).x);
                    m = warp_max(m);
                }
                float w = 0.f; // weight of this warp's part number `lane` of the eight
                if (lane < n) {
                    const float2 ml = pair(j0 + lane * split);
                    w = part_weight(ml.x, m);
                    l += ml.y * w;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float wk = __shfl_sync(0xffffffffu, w, j);
                    if (j >= n || !on || wk == 0.f) continue; // (an empty part's values were never written)
                    if (wide == 4) {
                        acc[0] += wk * x[j].x, acc[1] += wk * x[j].y, acc[2] += wk * x[j].z, acc[3] += wk * x[j].w;
                    } else {
                        const float *o = part(j0 + j * split) + (size_t)r * D + lane * 8;
                        const float4 y0 = *(const float4 *)o, y1 = *(const float4 *)(o + 4);
                        acc[0] += wk * y0.x, acc[1] += wk * y0.y, acc[2] += wk * y0.z, acc[3] += wk * y0.w;
                        acc[4] += wk * y1.x, acc[5] += wk * y1.y, acc[6] += wk * y1.z, acc[7] += wk * y1.w;
                    }
                }
            }
            l = warp_sum(l);
        }
        if (split > 1) { // the row's warps in order
            __syncthreads();
            if (on)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < wide) sm.acc[warp][lane * wide + e] = acc[e];
            if (lane == 0) sm.l[warp] = l;
            __syncthreads();
        }
        if (i >= n_rows || sub) continue;
        if (split > 1)
            for (int s = 1; s < split; ++s) {
                l += sm.l[warp + s];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < wide && on) acc[e] += sm.acc[warp + s][lane * wide + e];
            }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const int row = u.t * M + r;
        O *out = (O *)p.out + (u.r0 + row / p.group) * p.out_stride + ((long long)u.h * p.group + row % p.group) * D + lane * wide;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < wide && on) out[e] = out_from<O>(l == 0.f ? 0.f : acc[e] * inv);
    }
}

} // namespace ullm
