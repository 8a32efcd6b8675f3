// Attention of drafted rows over a paged cache with f32 queries: 32-bit products on the tensor cores.
//
// The formula is that of tree_attn.cu.  The tensor cores multiply 11-bit significands (tf32) and add in f32; a 32-bit value x is taken as the sum
// x = a + b of its 11 leading bits and the next 11, so that
//   x y = a a' + a b' + b a'  within  2^-22 + 2^-20 + 2^-21 of |x y|
// (what b of a query or a weight, b' of a key or value, and b b' leave out: the parts of the former are rounded, of the latter cut off, so that the largest
// values stay finite).  Below 2^-126 the parts have fewer bits; a block with a query or key beyond 2^60, where that could count, forms its
// products one by one.  Values of 16 bits fit in one part: two products instead of three.
// The tensor cores cut off what does not fit when they add, always towards zero, so that long sums come out too small: with a segment's weighted values left in their
// accumulators 1 to 4e-5 over 32,000 to 100,000 tokens.  They hold one block's sums only, which ordinary additions join to those of the blocks before (90 rows
// over heads of 64: 129 -> 132 us).  Errors against 64 bits, as a share of the values' mean: 1.4e-7 (root mean square) over 100,000 positive values, 9.4e-7 over such of either sign;
// the same formula in f32 with a matrix library: 1.4e-7 and 7.0e-7.
//
// A CTA of eight warps takes 16 or 32 query rows and walks blocks of 64 keys, whose keys and values arrive by cp.async, as they lie in the pages, while the
// block before is worked on.  A warp has 16 rows and a fixed share of every block's keys (8 or 16), keeps a maximum, a sum and weighted
// values for these keys alone, and the warps of a row meet once, at the end of the segment: there is no barrier between scores, softmax and weighted sums,
// and only the warps over the same keys wait for one another between blocks.
// The accumulators of the scores are in the place where the products with the values want the weights.  The order of a head's values, and of the keys, within a
// product is free as long as both sides agree; it is chosen so that a lane reads 16 neighbouring bytes.
// On the CUDA cores (tree_attn.cu) the reads of shared memory bound the same work: 32 lanes x 16 bytes take four cycles and feed 32 multiply-adds per lane.
// Rows are few (a group's heads x drafted tokens), so that tcgen05's tile of 128 rows would be empty for the most part.
// It is bound by chains of dependent instructions, eight or sixteen warps on an SM: issue slots 34 % and the tensor pipe 10 % busy for 24 units of 28 rows, 42 and 26 to 35 %
// for 90 rows; 32 sequences of one row and 1,500 keys (174 MB) 2.9 TB/s, 90 rows over heads of 64 29 TFLOP/s of 32-bit results, where the CUDA cores gave 2.6 TB/s
// and 14 to 16.
#include "engine.h"
#include "tree_sched.cuh"

#include <algorithm>

namespace ullm {
namespace {

constexpr int XT = 256, XK = 64;     // threads; keys of a block
constexpr float BIG = 1.152921504606847e18f; // 2^60
// places that a unit costs beside its blocks (90 rows over heads of 64: 1 and 3 for 135 us, 2 for 132; 32 sequences of one row: 60.5, 62.5 and 60.8); that a CTA takes at least
constexpr int X_COST = 2, X_MIN = 2;

template <typename KV, int D, int M> struct SplitCfg {
    static constexpr int RT = M / 16, KG = 8 / RT, NT = XK / KG / 8;   // row tiles; groups of keys; tiles of eight keys of a warp
    // bytes from key to key: lanes four apart read different banks
    static constexpr int KP = D * (int)sizeof(KV) + (sizeof(KV) == 4 ? 16 : 64), VP = D * (int)sizeof(KV) + 16;
    static constexpr int QF = M * D;                                   // floats of one part of the queries
    static constexpr int STAGE = XK * (KP + VP), SMEM = 2 * QF * (int)sizeof(float) + 2 * STAGE;
    static constexpr int PER_SM = D == 64 ? 2 : 1;                     // CTAs: 128 or 255 registers a thread
    static_assert(8 * 16 * D * (int)sizeof(float) <= 2 * STAGE, "the warps' results meet in the stages' memory");
};

// D += A B on 16 rows x 8 columns x 8 products
__device__ __forceinline__ void mma8(float (&d)[4], const float4 &a, float b0, float b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(__float_as_uint(a.x)), "r"(__float_as_uint(a.y)), "r"(__float_as_uint(a.z)), "r"(__float_as_uint(a.w)), "r"(__float_as_uint(b0)),
                   "r"(__float_as_uint(b1)));
}
// The 11 leading bits, rounded (the largest values become infinite) or cut off; x - cut11(x) is NaN for an infinity or a NaN
__device__ __forceinline__ float round11(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u); }
__device__ __forceinline__ float cut11(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// Eight neighbouring values as f32
__device__ __forceinline__ void widen8(float (&x)[8], const float *p) {
    const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void widen8(float (&x)[8], const __half *p) {
    const uint4 v = *(const uint4 *)p;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(*(const __half2 *)&w[i]);
        x[2 * i] = a.x, x[2 * i + 1] = a.y;
    }
}
__device__ __forceinline__ void widen8(float (&x)[8], const __nv_bfloat16 *p) {
    const uint4 v = *(const uint4 *)p;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
// acc[n] += (a + b) y[n] for several y of the cache, product by product, so that those into one place are apart; z: the sum of their squares.
// SETS: places per sum, 1 to 3
template <typename KV, int N, int SETS> __device__ __forceinline__ void products(float (&acc)[N][SETS][4], const float4 &a, const float4 &b, const float (&y0)[N], const float (&y1)[N], float &z) {
    if constexpr (sizeof(KV) == 4) {
        float h0[N], h1[N], l0[N], l1[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            h0[n] = cut11(y0[n]), h1[n] = cut11(y1[n]), l0[n] = y0[n] - h0[n], l1[n] = y1[n] - h1[n];
            z = fmaf(y0[n], y0[n], fmaf(y1[n], y1[n], z));
        }
#pragma unroll
        for (int n = 0; n < N; ++n) mma8(acc[n][SETS - 1], a, cut11(l0[n]), cut11(l1[n]));
#pragma unroll
        for (int n = 0; n < N; ++n) mma8(acc[n][SETS / 2], b, h0[n], h1[n]);
#pragma unroll
        for (int n = 0; n < N; ++n) mma8(acc[n][0], a, h0[n], h1[n]);
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n) z = fmaf(y0[n], y0[n], fmaf(y1[n], y1[n], z));
#pragma unroll
        for (int n = 0; n < N; ++n) mma8(acc[n][SETS - 1], b, y0[n], y1[n]);
#pragma unroll
        for (int n = 0; n < N; ++n) mma8(acc[n][0], a, y0[n], y1[n]);
    }
}

template <typename KV, int D, int M> __global__ void __launch_bounds__(XT, (SplitCfg<KV, D, M>::PER_SM)) tree_attn_split_kernel(const TreeDev p) {
    using C = SplitCfg<KV, D, M>;
    extern __shared__ __align__(16) uint8_t xsm[];
    float *const qa = (float *)xsm, *const qb = qa + C::QF; // the parts of the queries, as the products want them: 16 bytes per row tile, step and lane
    uint8_t *const stage0 = (uint8_t *)(qb + C::QF);
    __shared__ Seg seg;
    __shared__ int last;
    __shared__ long long offs[2][XK]; // where the keys of a block lie: bytes behind p.k and p.v, -1 for none
    __shared__ float2 ml[8][16];      // maximum and sum of each warp's rows
    pdl_wait_prior();
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rt = warp % C::RT, kg = warp / C::RT, kbase = kg * C::NT * 8;
    Sched<M, XK, X_COST, X_MIN> sched(p);
    const bool some = warp == 0 && sched.init();
    // The warps over the same keys fetch them and wait for one another, and for no others.
    constexpr int PIECES = D * (int)sizeof(KV) / 16, TG = 32 * C::RT, STEP = TG / PIECES; // 16-byte pieces of a row; threads of such a group; rows that they take at once
    const int tg = rt * 32 + lane, piece_j = tg / PIECES, piece_c = tg % PIECES * 16;
    auto meet = [&] {
        if constexpr (C::RT == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + kg), "n"(TG) : "memory");
    };
    for (;;) {
        __syncthreads();
        if (warp == 0) {
            Seg next;
            next.count = 0;
            if (some) next = sched.next(nullptr);
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
        const int *const table = p.blocks + (size_t)v.id * p.max_blocks;
        auto entry = [&](int token) { return p.page_log >= 0 ? token >> p.page_log : token / p.page_size; };
        auto page_at = [&](int token) { return token < key_end ? table[entry(token)] : -1; };
        auto place = [&](int page, int token) { // a key behind the last, or of a page outside the pool, has none
            return (unsigned)page < (unsigned)p.n_pages ? (page * p.page_stride + (token - entry(token) * p.page_size) * p.slot_stride + w.h * p.head_stride) * (long long)sizeof(KV) : -1ll;
        };
        auto fetch = [&](int blk, uint8_t *stage) { // zeros for a key that has no place
            const long long *const at = offs[(blk - w.blk) & 1];
#pragma unroll
            for (int j0 = 0; j0 < C::NT * 8; j0 += STEP) {
                const int j = kbase + j0 + piece_j;
                const long long off = at[j];
                const bool on = off >= 0;
                const long long from = on ? off + piece_c : 0;
                copy16(stage + j * C::KP + piece_c, p.k + from, on);
                copy16(stage + XK * C::KP + j * C::VP + piece_c, p.v + from, on);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        const bool mine = tg < C::NT * 8; // threads that look up a key each
        auto begin = [&] {
            if (mine) { // keys of the first two blocks
                const int key = w.blk * XK + kbase + tg, page0 = page_at(key), page1 = page_at(key + XK);
                offs[0][kbase + tg] = place(page0, key), offs[1][kbase + tg] = place(page1, key + XK);
            }
            meet();
            fetch(w.blk, stage0);
        };
        begin();
        const bool work = rt * 16 < rows;
        for (int i = tid; i < M * (D / 4); i += XT) { // queries: value 8 t + e of 32 is product t (or t + 4, for e >= 4) of step e % 4
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) x = *(const float4 *)((const float *)p.q + (v.r0 + token_of(r)) * p.q_stride + (long long)head_of(r) * D + d);
            const float y[4] = {x.x, x.y, x.z, x.w};
            const int step = d / 32 * 4, l = r % 8 * 4 + d % 32 / 8, at = (((r / 16) * (D / 8) + step) * 32 + l) * 4 + (r % 16 / 8 + d % 8 / 4 * 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float a = round11(y[e]), b = round11(y[e] - a);
                if (!(fabsf(y[e]) <= BIG)) seg.big = 1, a = y[e], b = 0.f; // infinities and NaN too
                qa[at + e * 128] = a, qb[at + e * 128] = b;
            }
        }
        __syncthreads();
        const bool big = seg.big;
        const int row[2] = {rt * 16 + g, rt * 16 + g + 8}, token[2] = {token_of(row[0]), token_of(row[1])};
        float m[2], l[2]; // l: this lane's share
        float o[D / 32][4][1][4]; // [c][i]: value 32 c + 8 t + i of rows 0 and 1 in 0 and 2, value 32 c + 8 t + 4 + i in 1 and 3
        // Values that are not finite must not reach a row that does not see them (0 * inf), nor be split.  They show in the sums, and the segment is
        // worked through again with a look at every value: looking the first time cost 5 % (90 rows).
        for (bool careful = false;;) {
            m[0] = m[1] = -INFINITY, l[0] = l[1] = 0.f;
#pragma unroll
            for (int n = 0; n < D / 2; ++n) o[n / 16][n / 4 % 4][0][n % 4] = 0.f;
            for (int blk = w.blk; blk < blk_end; ++blk) {
                uint8_t *const ks = stage0 + ((blk - w.blk) & 1) * C::STAGE, *const vs = ks + XK * C::KP;
                const int k0 = blk * XK;
                if (blk + 1 < blk_end) {
                    fetch(blk + 1, stage0 + ((blk + 1 - w.blk) & 1) * C::STAGE);
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                } else {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                }
                meet();
                // the block after the next: its page numbers travel while this one is worked on
                const int ahead = (blk + 2) * XK + kbase + tg;
                const bool more = mine && blk + 2 < blk_end;
                const int page = more ? page_at(ahead) : -1;
                if (work && k0 + kbase < key_end) {
                    constexpr int SETS = C::NT == 1 ? 3 : 2; // a product waits for the one before it in its place: three places at least
                    float parts[C::NT][SETS][4], s[C::NT][4], z = 0.f;
#pragma unroll
                    for (int n = 0; n < C::NT; ++n)
#pragma unroll
                        for (int e = 0; e < SETS * 4; ++e) parts[n][e / 4][e % 4] = 0.f;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) { // (90 rows over heads of 64: 132 us, 136 with a loop; over heads of 128: 159 us, 164 with one)
                        float y[C::NT][8];
#pragma unroll
                        for (int n = 0; n < C::NT; ++n) widen8(y[n], (const KV *)(ks + (kbase + n * 8 + g) * C::KP) + c * 32 + t * 8);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = ((rt * (D / 8) + c * 4 + i) * 32 + lane) * 4;
                            const float4 a = *(const float4 *)(qa + at);
                            const float4 b = *(const float4 *)(qb + at);
                            float y0[C::NT], y1[C::NT];
#pragma unroll
                            for (int n = 0; n < C::NT; ++n) y0[n] = y[n][i], y1[n] = y[n][4 + i];
                            products<KV>(parts, a, b, y0, y1, z);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < C::NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[n][e] = parts[n][0][e];
#pragma unroll
                            for (int k = 1; k < SETS; ++k) s[n][e] += parts[n][k][e];
                        }
                    if (__any_sync(0xffffffffu, !(z < BIG * BIG)) || big) { // (b times an infinity is not what x times it is, either)
#pragma unroll
                        for (int n = 0; n < C::NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const KV *const key = (const KV *)(ks + (kbase + n * 8 + 2 * t + (e & 1)) * C::KP);
                                float sum = 0.f;
                                for (int d = 0; d < D; ++d) {
                                    const int at = ((rt * (D / 8) + d / 32 * 4 + d % 4) * 32 + g * 4 + d % 32 / 8) * 4 + (e >> 1) + d % 8 / 4 * 2;
                                    sum = fmaf(qa[at] + qb[at], (float)key[d], sum);
                                }
                                s[n][e] = sum;
                            }
                    }
                    const bool all = k0 + kbase + C::NT * 8 <= min(key_end, v.ctx); // every row sees all of them
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int n = 0; n < C::NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[n][e] *= p.scale_log2;
                            if (!all) {
                                const int key = k0 + kbase + n * 8 + 2 * t + (e & 1);
                                bool see = key < key_end && row[e >> 1] < rows;
                                if (see && key >= v.ctx) see = sees(p, v, token[e >> 1], key - v.ctx);
                                if (!see) s[n][e] = -INFINITY;
                            }
                            mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
                        }
                    float corr[2];
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        mx[a] = fmaxf(mx[a], __shfl_xor_sync(0xffffffffu, mx[a], 1));
                        mx[a] = fmaxf(fmaxf(mx[a], __shfl_xor_sync(0xffffffffu, mx[a], 2)), m[a]);
                        corr[a] = m[a] == -INFINITY ? 0.f : exp2f(m[a] - mx[a]);
                        m[a] = mx[a], l[a] *= corr[a];
                    }
                    // nothing seen so far: all weights are zero.  (A score of +inf or NaN gives NaN, as the formula does.)
#pragma unroll
                    for (int n = 0; n < C::NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[n][e] = s[n][e] == -INFINITY ? 0.f : exp2f(s[n][e] - m[e >> 1]);
                            l[e >> 1] += s[n][e];
                        }
                    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                        for (int n = 0; n < D / 2; ++n) o[n / 16][n / 4 % 4][0][n % 4] *= corr[n % 4 / 2];
                    }
                    // Values that are not finite become zeros here and are added at the end.
                    if (careful) {
                        KV *const own = (KV *)(vs + kbase * C::VP);
                        float bad = 0.f;
#pragma unroll 2
                        for (int i = lane; i < C::NT * 8 * (D / 8); i += 32) {
                            float y[8];
                            widen8(y, (const KV *)((uint8_t *)own + i / (D / 8) * C::VP) + i % (D / 8) * 8);
#pragma unroll
                            for (int e = 0; e < 8; ++e) bad = fmaf(y[e], 0.f, bad);
                        }
                        if (__any_sync(0xffffffffu, bad != bad)) {
                            for (int i = lane; i < C::NT * 8 * D; i += 32) {
                                KV *const at = (KV *)((uint8_t *)own + i / D * C::VP) + i % D;
                                if (!isfinite((float)*at)) *at = (KV)0.f;
                            }
                            seg.odd = 1;
                            __syncwarp();
                        }
                    }
                    float4 a[C::NT], b[C::NT];
#pragma unroll
                    for (int n = 0; n < C::NT; ++n) {
                        const float4 x = make_float4(s[n][0], s[n][2], s[n][1], s[n][3]); // product t is key 2 t, product t + 4 key 2 t + 1
                        a[n] = make_float4(round11(x.x), round11(x.y), round11(x.z), round11(x.w));
                        b[n] = make_float4(round11(x.x - a[n].x), round11(x.y - a[n].y), round11(x.z - a[n].z), round11(x.w - a[n].w));
                    }
                    float unused = 0.f;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float sum[4][1][4]; // of this block
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum[i / 4][0][i % 4] = 0.f;
#pragma unroll
                        for (int n = 0; n < C::NT; ++n) {
                            const KV *const v0 = (const KV *)(vs + (kbase + n * 8 + 2 * t) * C::VP) + g * 4 + c * 32, *const v1 = (const KV *)((const uint8_t *)v0 + C::VP);
                            const float4 y0 = widen4(v0), y1 = widen4(v1);
                            const float w0[4] = {y0.x, y0.y, y0.z, y0.w}, w1[4] = {y1.x, y1.y, y1.z, y1.w};
                            products<KV>(sum, a[n], b[n], w0, w1, unused);
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[c][i / 4][0][i % 4] += sum[i / 4][0][i % 4];
                    }
                }
                if (more) offs[(blk - w.blk) & 1][kbase + tg] = place(page, ahead);
                meet(); // the stage is free
            }
            bool odd = false;
            if (work && !careful)
#pragma unroll
                for (int n = 0; n < D / 2; ++n) odd |= !(fabsf(o[n / 16][n / 4 % 4][0][n % 4]) < INFINITY);
            if (!__syncthreads_or(odd)) break;
            careful = true;
            begin();
        }
        // the warps' results meet in the stages' memory
        float *const red = (float *)stage0;
        if (work) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                float sum = l[a];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (t == 0) ml[warp][g + 8 * a] = make_float2(m[a], sum);
                float *const to = red + (warp * 16 + g + 8 * a) * D + t * 8;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    *(float4 *)(to + c * 32) = make_float4(o[c][0][0][2 * a], o[c][1][0][2 * a], o[c][2][0][2 * a], o[c][3][0][2 * a]);
                    *(float4 *)(to + c * 32 + 4) = make_float4(o[c][0][0][2 * a + 1], o[c][1][0][2 * a + 1], o[c][2][0][2 * a + 1], o[c][3][0][2 * a + 1]);
                }
            }
        }
        __syncthreads();
        const bool whole = w.flags & 1, odd = seg.odd;
        float *const to = whole ? nullptr : part_of<M>(p, blockIdx.x, w.flags >> 1);
        for (int i = tid; i < rows * (D / 4); i += XT) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < C::KG; ++k) top = fmaxf(top, ml[k * C::RT + r / 16][r % 16].x);
#pragma unroll
            for (int k = 0; k < C::KG; ++k) {
                const int wp = k * C::RT + r / 16;
                const float2 a = ml[wp][r % 16];
                const float c = a.x == -INFINITY ? 0.f : exp2f(a.x - top);
                const float4 y = *(const float4 *)(red + (wp * 16 + r % 16) * D + d);
                sum += a.y * c; // (NaN where a score was NaN)
                x.x += c * y.x, x.y += c * y.y, x.z += c * y.z, x.w += c * y.w;
            }
            if (odd) { // infinities and NaN of the tokens that the row does see
                const int last = min(key_end, blk_end * XK), me = token_of(r);
                for (int key = w.blk * XK; key < last; ++key) {
                    const int page = table[key / p.page_size];
                    if ((unsigned)page >= (unsigned)p.n_pages || (key >= v.ctx && !sees(p, v, me, key - v.ctx))) continue;
                    const long long at = page * p.page_stride + key % p.page_size * p.slot_stride + w.h * p.head_stride;
                    const float4 y = widen4((const KV *)p.v + at + d);
                    if (isfinite(y.x) && isfinite(y.y) && isfinite(y.z) && isfinite(y.w)) continue;
                    const bool none = has_no_weight((const float *)p.q + (v.r0 + me) * p.q_stride + (long long)head_of(r) * D, (const KV *)p.k + at, D, p.scale_log2);
                    if (!isfinite(y.x)) x.x += none ? NAN : y.x;
                    if (!isfinite(y.y)) x.y += none ? NAN : y.y;
                    if (!isfinite(y.z)) x.z += none ? NAN : y.z;
                    if (!isfinite(y.w)) x.w += none ? NAN : y.w;
                }
            }
            if (whole) {
                const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                const float4 y = sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                *(float4 *)((float *)p.out + (v.r0 + token_of(r)) * p.out_stride + (long long)head_of(r) * D + d) = y;
            } else {
                *(float4 *)(to + (size_t)r * D + d) = x;
                if (d == 0) *(float2 *)(to + (size_t)M * D + 2 * r) = make_float2(top, sum);
            }
        }
        if (!whole) join_last<float, M, D>(p, w, &last);
    }
}

// Zeros in front of a call: the work area may hold anything.  (32-bit cache 19.5 us; with counts that carried the number of their call, in memory that was left as it
// was, 21.5, and numbers of that size in the memory were taken for counts.)
__global__ void tree_count_kernel(int *count, int n) {
    pdl_wait_prior();
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < n; i += blockDim.x) count[i] = 0;
}

template <typename KV, int D, int M> cudaError_t launch_as(const DeviceInfo &dev, const TreeDev &t, bool pdl, cudaStream_t st) {
    using C = SplitCfg<KV, D, M>;
    cudaError_t e = cudaFuncSetAttribute(tree_attn_split_kernel<KV, D, M>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    const int ctas = dev.sm_count * C::PER_SM;
    if ((e = launch_kernel(tree_count_kernel, dim3(1), dim3(XT), 0, st, pdl, t.count, ctas)) != cudaSuccess) return e;
    return launch_kernel(tree_attn_split_kernel<KV, D, M>, dim3(ctas), dim3(XT), (size_t)C::SMEM, st, pdl, t);
}
template <typename KV, int D> cudaError_t launch_for(const DeviceInfo &dev, const TreeDev &t, bool pdl, cudaStream_t st) {
    // Rows per sequence and key head on average (the lengths themselves are on the device; either way is right for any of them).
    const long long rows = ((long long)t.n_rows * t.group + t.n_seq - 1) / t.n_seq;
    // Tiles of 32 rows split the keys half as often (90 rows over heads of 64: 132 us, with 16 rows 162; 64 rows took 7 % longer than 32), but 16 rows spread a little work over more CTAs, where
    // even tables in full use would give a CTA no more than four blocks (24 units of 28 rows and up to 2,000 keys: 19.5 us, with 32 rows 22.1; 32 sequences of one row: 60.7 and 67.9).
    const long long blocks = (rows + 31) / 32 * t.n_seq * t.n_kv * (((long long)t.max_blocks * t.page_size + XK - 1) / XK);
    if (rows <= 16 || blocks <= 4 * dev.sm_count * SplitCfg<KV, D, 16>::PER_SM) return launch_as<KV, D, 16>(dev, t, pdl, st);
    return launch_as<KV, D, 32>(dev, t, pdl, st);
}
template <typename KV> cudaError_t launch_dim(const DeviceInfo &dev, const TreeDev &t, bool pdl, cudaStream_t st) {
    return t.dim == 64 ? launch_for<KV, 64>(dev, t, pdl, st) : launch_for<KV, 128>(dev, t, pdl, st);
}

} // namespace

bool tree_attn_split_supported(int dim) { return dim == 64 || dim == 128; }

cudaError_t launch_tree_attn_split(const DeviceInfo &dev, int kv_dtype, const TreeDev &t, bool pdl, cudaStream_t st) {
    if (kv_dtype == ULLM_DTYPE_F32) return launch_dim<float>(dev, t, pdl, st);
    return kv_dtype == ULLM_DTYPE_F16 ? launch_dim<__half>(dev, t, pdl, st) : launch_dim<__nv_bfloat16>(dev, t, pdl, st);
}

} // namespace ullm
