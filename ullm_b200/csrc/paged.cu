// Tables of a paged key/value cache, the plan of a step of drafted trees, and the pass that normalises, rotates and
// stores a step's projections.  The rules are in include/ullm_cuda.h.
//
// Everything the tables hang on - lengths, page numbers, reference counts - is read and written on the device, so a
// speculative step (grow, layers, accept) needs no host round trip and can be captured once and replayed.  There is no
// list of free pages: a page is free when its count is zero, and kv_grow hands out the lowest-numbered ones in
// list order, so that the result does not depend on the order in which pages were given back.
#include "paged.h"
#include "engine.h"

#include <algorithm>
#include <cstdint>
#include <type_traits>

namespace ullm {

const char *pool_check(const ullm_kv_pages *kv, PoolDev *out) {
    if (kv->dtype != ULLM_DTYPE_F32 && kv->dtype != ULLM_DTYPE_F16 && kv->dtype != ULLM_DTYPE_BF16) return "pages hold f32, f16 or bf16 values";
    if (!kv->n_layer || !kv->n_pages || !kv->page_size || !kv->n_kv_head || !kv->head_dim) return "a pool has at least one layer, page, slot, head and value";
    if (kv->head_dim % 8 || kv->head_dim > 256) return "head_dim must be a multiple of 8, at most 256";
    if (kv->n_pages > INT32_MAX / 2 || kv->page_size > 65536 || kv->n_layer > 32767 || kv->n_kv_head > 65535) return "pool dimension too large";
    const size_t eb = dtype_bytes(kv->dtype), per16 = 16 / eb;
    if ((uintptr_t)kv->d_k % 16 || (uintptr_t)kv->d_v % 16) return "d_k and d_v must be 16-byte aligned";
    const size_t strides[4] = {kv->layer_stride, kv->page_stride, kv->slot_stride, kv->head_stride};
    const size_t counts[4] = {kv->n_layer, kv->n_pages, kv->page_size, kv->n_kv_head};
    for (int i = 0; i < 4; ++i) {
        if (strides[i] % per16) return "pool strides must be multiples of 16 bytes";
        if (counts[i] > 1 && strides[i] < kv->head_dim) return "pool strides must be at least head_dim";
        if (strides[i] > ((size_t)1 << 39) / eb) return "pool stride too large";
    }
    out->k = (uint8_t *)kv->d_k, out->v = (uint8_t *)kv->d_v;
    out->layer_stride = (long long)kv->layer_stride, out->page_stride = (long long)kv->page_stride;
    out->slot_stride = (long long)kv->slot_stride, out->head_stride = (long long)kv->head_stride;
    out->n_layer = (int)kv->n_layer, out->n_pages = (int)kv->n_pages, out->page_size = (int)kv->page_size;
    out->n_kv_head = (int)kv->n_kv_head, out->head_dim = (int)kv->head_dim, out->elem_bytes = (int)eb;
    return nullptr;
}

namespace {

__device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ void set_fault(int *fault, int bits) {
    if (fault && bits) atomicOr(fault, bits);
}

// Whether a row of the table can hold `len` tokens.  (Asked before `len` is counted in pages: near the end of the range that sum would pass 32 bits.)
__device__ __forceinline__ bool len_fits(const TableDev &t, int page_size, int len) { return len >= 0 && len <= (long long)t.max_blocks * page_size; }

// Whether `v` occurs in list[0 .. n) at another place than `self`; every thread of the CTA calls it with the same arguments.
__device__ __forceinline__ bool cta_listed_elsewhere(const int *list, int n, int v, int self) {
    bool hit = false;
    for (int j = threadIdx.x; j < n; j += blockDim.x) hit |= j != self && list[j] == v;
    return __syncthreads_or(hit) != 0;
}

// ---- fork: one CTA per pair ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) kv_fork_kernel(const TableDev t, int page_size, int n_pages, const int *src, const int *dst, int n) {
    pdl_wait_prior();
    pdl_launch_dependents();
    const int i = blockIdx.x, s = src[i], d = dst[i];
    int bad = 0, len = 0, blocks = 0;
    if (s < 0 || s >= t.n_seq || d < 0 || d >= t.n_seq || s == d) bad = ULLM_KV_FAULT_SEQ;
    // a row that is written here is read by no other pair and written by no other pair
    if (cta_listed_elsewhere(dst, n, d, i) || cta_listed_elsewhere(src, n, d, -1)) bad |= ULLM_KV_FAULT_SEQ;
    if (!bad) {
        len = t.len[s];
        if (!len_fits(t, page_size, len)) bad = ULLM_KV_FAULT_LEN;
        else if (t.len[d] != 0) bad = ULLM_KV_FAULT_SEQ;
        else blocks = cdiv(len, page_size);
    }
    const int *from = t.blocks + (size_t)(bad ? 0 : s) * t.max_blocks;
    bool out = false;
    if (!bad)
        for (int j = threadIdx.x; j < blocks; j += blockDim.x) out |= (unsigned)from[j] >= (unsigned)n_pages;
    if (__syncthreads_or(out)) bad |= ULLM_KV_FAULT_PAGE;
    if (bad) {
        if (threadIdx.x == 0) set_fault(t.fault, bad);
        return;
    }
    int *to = t.blocks + (size_t)d * t.max_blocks;
    for (int j = threadIdx.x; j < blocks; j += blockDim.x) {
        const int page = from[j];
        to[j] = page;
        atomicAdd(t.refs + page, 1);
    }
    if (threadIdx.x == 0) t.len[d] = len;
}

// ---- trim and the second half of accept: one CTA per sequence -------------------------------------------------------
// Gives back blocks [keep, have) of a row; every thread of the CTA calls it.
__device__ __forceinline__ void release_blocks(const TableDev &t, int seq, int keep, int have, int n_pages) {
    const int *row = t.blocks + (size_t)seq * t.max_blocks;
    int bad = 0;
    for (int j = keep + threadIdx.x; j < have; j += blockDim.x) {
        const int page = row[j];
        if ((unsigned)page >= (unsigned)n_pages) {
            bad = ULLM_KV_FAULT_PAGE;
        } else if (atomicSub(t.refs + page, 1) <= 0) { // more owners gave it back than there were
            atomicAdd(t.refs + page, 1);
            bad = ULLM_KV_FAULT_PAGE;
        }
    }
    set_fault(t.fault, bad);
}

__global__ void __launch_bounds__(128) kv_trim_kernel(const TableDev t, int page_size, int n_pages, const int *seq, const int *new_len, int n) {
    pdl_wait_prior();
    pdl_launch_dependents();
    const int i = blockIdx.x, s = seq[i];
    int bad = s < 0 || s >= t.n_seq ? ULLM_KV_FAULT_SEQ : 0;
    if (cta_listed_elsewhere(seq, n, s, i)) bad |= ULLM_KV_FAULT_SEQ;
    int len = 0, want = 0;
    if (!bad) {
        len = t.len[s], want = new_len ? new_len[i] : 0;
        if (want < 0 || want > len || !len_fits(t, page_size, len)) bad = ULLM_KV_FAULT_LEN;
    }
    __syncthreads(); // every thread has read the length before it changes
    if (bad) {
        if (threadIdx.x == 0) set_fault(t.fault, bad);
        return;
    }
    release_blocks(t, s, cdiv(want, page_size), cdiv(len, page_size), n_pages);
    if (threadIdx.x == 0) t.len[s] = want;
}

// ---- accept ---------------------------------------------------------------------------------------------------------
// grid (sequences, Y): CTA (i, y) moves the kept rows of its share of the layers' K and V.  A thread owns 16-byte pieces of a row and
// takes up to eight rows into registers before it stores them: kept indices increase, so a row is never moved onto one that a
// later batch still reads (destination j <= path[j] < path[j + 1]), and pieces of different threads never meet.  The
// verdict on the entry is the same in every CTA (the tables do not change until kv_accept_end_kernel); the first one leaves it
// in t.work[i].  What costs time is the chain of loads in front of the first move (entry, length, path, page numbers,
// counts): Y is chosen so that all CTAs run at once and pay it once (192 entries, 24 matrices: 21 us with a CTA for each matrix).
constexpr int MOVE_BATCH = 8, MOVE_KEEP = 64; // MOVE_KEEP: rows whose places a CTA keeps in shared memory
__global__ void __launch_bounds__(128) kv_accept_move_kernel(const TableDev t, const PoolDev pool, const int *seq, const int *draft, const int *path,
                                                            const int *kept, int n, int max_path) {
    __shared__ long long s_from[MOVE_KEEP], s_to[MOVE_KEEP]; // bytes from a matrix' start
    __shared__ int s_first;                                  // rows of the path that stay where they are
    pdl_wait_prior();
    pdl_launch_dependents();
    const int i = blockIdx.x, s = seq[i], nd = draft[i], nk = kept[i], ps = pool.page_size;
    const int *p = path + (size_t)i * max_path;
    int bad = s < 0 || s >= t.n_seq ? ULLM_KV_FAULT_SEQ : 0;
    if (threadIdx.x == 0) s_first = INT32_MAX;
    if (cta_listed_elsewhere(seq, n, s, i)) bad |= ULLM_KV_FAULT_SEQ;
    int len = 0;
    if (!bad) {
        len = t.len[s];
        if (nd < 0 || nd > len || nk < 0 || nk > nd || nk > max_path || !len_fits(t, ps, len)) bad = ULLM_KV_FAULT_LEN;
    }
    const int base = len - nd;
    const int *row = t.blocks + (size_t)(bad ? 0 : s) * t.max_blocks;
    auto at = [&](int token, int page) { return (page * pool.page_stride + (token % ps) * pool.slot_stride) * pool.elem_bytes; };
    int seen = 0;
    if (!bad)
        for (int j = threadIdx.x; j < nk; j += blockDim.x) {
            const int from = p[j];
            if (from < 0 || from >= nd || (j > 0 && from <= p[j - 1])) {
                seen |= ULLM_KV_FAULT_PATH;
            } else if (from != j) {
                const int a = row[(base + from) / ps], b = row[(base + j) / ps];
                if ((unsigned)a >= (unsigned)pool.n_pages || (unsigned)b >= (unsigned)pool.n_pages) seen |= ULLM_KV_FAULT_PAGE;
                else if (t.refs[b] != 1) seen |= ULLM_KV_FAULT_SHARED;
                if (j < MOVE_KEEP) s_from[j] = at(base + from, a), s_to[j] = at(base + j, b);
                atomicMin(&s_first, j);
            }
        }
    if (__syncthreads_or(seen)) {
        set_fault(t.fault, seen);
        bad |= ULLM_KV_FAULT_PATH; // whichever it was, a thread that saw it has reported it
    } else if (bad && threadIdx.x == 0) {
        set_fault(t.fault, bad);
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) t.work[i] = bad;
    const int first = s_first;
    if (bad || first >= nk) return;
    auto from_at = [&](int j) { return j < MOVE_KEEP ? s_from[j] : at(base + p[j], row[(base + p[j]) / ps]); };
    auto to_at = [&](int j) { return j < MOVE_KEEP ? s_to[j] : at(base + j, row[(base + j) / ps]); };
    const int pieces = pool.head_dim * pool.elem_bytes / 16, per = pieces * pool.n_kv_head, mats = 2 * pool.n_layer;
    const int m0 = (int)((long long)mats * blockIdx.y / gridDim.y), m1 = (int)((long long)mats * (blockIdx.y + 1) / gridDim.y);
    for (int c = threadIdx.x; c < per * (m1 - m0); c += blockDim.x) {
        const int mat = m0 + c / per, r = c % per;
        uint8_t *const col = (mat & 1 ? pool.v : pool.k) +
                             ((mat >> 1) * pool.layer_stride + (long long)(r / pieces) * pool.head_stride) * pool.elem_bytes + (r % pieces) * 16;
        for (int j = first; j < nk; j += MOVE_BATCH) { // from the first row that moves on, every one does
            uint4 v[MOVE_BATCH];
#pragma unroll
            for (int u = 0; u < MOVE_BATCH; ++u)
                if (j + u < nk) v[u] = *(const uint4 *)(col + from_at(j + u));
#pragma unroll
            for (int u = 0; u < MOVE_BATCH; ++u)
                if (j + u < nk) *(uint4 *)(col + to_at(j + u)) = v[u];
        }
    }
}
__global__ void __launch_bounds__(128) kv_accept_end_kernel(const TableDev t, int page_size, int n_pages, const int *seq, const int *draft, const int *kept) {
    pdl_wait_prior();
    pdl_launch_dependents();
    const int i = blockIdx.x;
    if (t.work[i]) return;
    const int s = seq[i], len = t.len[s], want = len - draft[i] + kept[i];
    __syncthreads();
    release_blocks(t, s, cdiv(want, page_size), cdiv(len, page_size), n_pages);
    if (threadIdx.x == 0) t.len[s] = want;
}

// ---- grow -----------------------------------------------------------------------------------------------------------
// Exclusive prefix sum over the CTA's 1024 threads; returns the sum of all.  Sums stop at SCAN_MAX, more than any pool has pages: what many long
// rows ask for together passes 32 bits.
constexpr unsigned SCAN_MAX = 1u << 30;
__device__ __forceinline__ int cta_scan1024(int v, int *excl, int *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto add = [](unsigned a, unsigned b) { return min(a + b, SCAN_MAX); };
    unsigned x = min((unsigned)v, SCAN_MAX);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x = add(x, y);
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = (int)x;
    __syncthreads();
    if (warp == 0) {
        unsigned w = (unsigned)warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w = add(w, y);
        }
        warp_sums[lane] = (int)w;
    }
    __syncthreads();
    *excl = (int)x - v + (warp ? warp_sums[warp - 1] : 0); // (of no use once the sum has stopped)
    return warp_sums[31];
}

// Work area of kv_grow: per entry the place of its first page in the list of picked ones, its need (| copy flag) and
// its copy {from, to, slots}; per table row how often it is listed; then the picked pages.
__host__ __device__ constexpr size_t grow_work_ints(size_t n_pages, size_t n_seq) { return 6 * n_seq + n_pages + 16; }

// One CTA: lengths -> needs -> the lowest free pages -> tables.  Reads before writes throughout: needs and copies are
// decided on the counts as they were before the call.
constexpr int FIRST_MAX = 2048; // entries whose places are searched in shared memory
__global__ void __launch_bounds__(1024) kv_grow_plan_kernel(const TableDev t, int page_size, int n_pages, const int *seq, const int *add, int n) {
    __shared__ int sums[32], s_first[FIRST_MAX];
    pdl_wait_prior();
    pdl_launch_dependents();
    const int tid = threadIdx.x;
    int *const first = t.work, *const need = first + t.n_seq, *const copy = need + t.n_seq, *const listed = copy + 3 * t.n_seq,
        *const picked = listed + t.n_seq;
    constexpr int COW = 1 << 30;
    for (int i = tid; i < n; i += 1024)
        if (seq[i] >= 0 && seq[i] < t.n_seq) listed[seq[i]] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += 1024)
        if (seq[i] >= 0 && seq[i] < t.n_seq) atomicAdd(listed + seq[i], 1);
    __syncthreads();
    long long total = 0;
    for (int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + tid;
        int want = 0, flag = 0;
        if (i < n) {
            const int s = seq[i], a = add[i];
            int bad = s < 0 || s >= t.n_seq || listed[s] != 1 ? ULLM_KV_FAULT_SEQ : 0;
            if (!bad) {
                const int len = t.len[s];
                const long long end = (long long)len + a;
                if (len < 0 || a < 0 || end > (long long)t.max_blocks * page_size) {
                    bad = ULLM_KV_FAULT_LEN;
                } else {
                    if (a > 0 && len % page_size) {
                        const int last = t.blocks[(size_t)s * t.max_blocks + len / page_size];
                        if ((unsigned)last >= (unsigned)n_pages) bad = ULLM_KV_FAULT_PAGE;
                        else if (t.refs[last] > 1) flag = COW;
                    }
                    want = cdiv((int)end, page_size) - cdiv(len, page_size) + (flag ? 1 : 0);
                }
            }
            if (bad) {
                set_fault(t.fault, bad);
                want = -1;
            }
            copy[3 * i] = -1;
        }
        int excl;
        const int sum = cta_scan1024(want > 0 ? want : 0, &excl, sums);
        if (i < n) {
            const int f = (int)min(total + excl, (long long)INT32_MAX / 2);
            need[i] = want < 0 ? -1 : want | flag, first[i] = f;
            if (i < FIRST_MAX) s_first[i] = f;
        }
        total += sum;
    }
    // the lowest `total` pages that nobody uses, in order: 8 counts per thread and sweep
    if (total > n_pages) {
        if (tid == 0) set_fault(t.fault, ULLM_KV_FAULT_NO_PAGES);
        return;
    }
    int found = 0;
    for (int p0 = 0; p0 < n_pages && found < total; p0 += 8192) {
        const int at = p0 + tid * 8;
        unsigned bits = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (at + u < n_pages && t.refs[at + u] == 0) bits |= 1u << u;
        int excl;
        const int sum = cta_scan1024(__popc(bits), &excl, sums);
        int r = found + excl;
        for (; bits; bits &= bits - 1, ++r)
            if (r < total) picked[r] = at + __ffs(bits) - 1;
        found += sum;
    }
    if (found < total) {
        if (tid == 0) set_fault(t.fault, ULLM_KV_FAULT_NO_PAGES);
        return;
    }
    __syncthreads();
    // hand them out: page u of the list belongs to the last entry whose first page is not behind u and that needs any
    for (int u = tid; u < (int)total; u += 1024) {
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if ((mid < FIRST_MAX ? s_first[mid] : first[mid]) <= u) lo = mid;
            else hi = mid;
        }
        const int i = lo, s = seq[i], len = t.len[s], k = u - (i < FIRST_MAX ? s_first[i] : first[i]);
        const bool cow = (need[i] & COW) != 0;
        const int b = cdiv(len, page_size) - (cow ? 1 : 0) + k, page = picked[u];
        int *const e = t.blocks + (size_t)s * t.max_blocks + b;
        if (cow && k == 0) {
            const int old = *e;
            atomicSub(t.refs + old, 1);
            copy[3 * i] = old, copy[3 * i + 1] = page, copy[3 * i + 2] = len % page_size;
        }
        *e = page;
        t.refs[page] = 1;
    }
    __syncthreads();
    for (int i = tid; i < n; i += 1024)
        if (need[i] >= 0) t.len[seq[i]] += add[i];
}

// ---- copies of whole pages ------------------------------------------------------------------------------------------
// Slots [0, slots) of page `from` to page `to` in the CTA's share of the layers' K and V (blockIdx.y of gridDim.y).  A thread's 16-byte pieces are
// 256 apart; their places (slot, head, piece) are counted on, not divided out, and a piece goes as far as every other one (192 half pages in 24
// matrices, a CTA each and a division for every digit: 34 us, 76 % of the issue slots; nine CTAs per entry, places
// counted on: 21 us).
__device__ __forceinline__ void copy_slots(const PoolDev &pool, int from, int to, int slots) {
    const int pieces = pool.head_dim * pool.elem_bytes / 16, heads = pool.n_kv_head, mats = 2 * pool.n_layer;
    const int m0 = (int)((long long)mats * blockIdx.y / gridDim.y), m1 = (int)((long long)mats * (blockIdx.y + 1) / gridDim.y);
    const long long slot_b = pool.slot_stride * pool.elem_bytes, head_b = pool.head_stride * pool.elem_bytes;
    const long long start = from * pool.page_stride * pool.elem_bytes, way = (to - from) * pool.page_stride * pool.elem_bytes;
    const int step_p = 256 % pieces, step_h = 256 / pieces % heads, step_s = 256 / pieces / heads, tid = threadIdx.x;
    const int p0 = tid % pieces, h0 = tid / pieces % heads, s0 = tid / pieces / heads;
    for (int m = m0; m < m1; ++m) {
        uint8_t *const mem = (m & 1 ? pool.v : pool.k) + (m >> 1) * pool.layer_stride * pool.elem_bytes + start;
        int p = p0, h = h0, s = s0;
        while (s < slots) { // eight loads in flight per thread
            uint4 v[8];
            uint8_t *at[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                at[u] = s < slots ? mem + s * slot_b + h * head_b + p * 16 : nullptr;
                p += step_p, h += step_h, s += step_s;
                if (p >= pieces) p -= pieces, ++h;
                if (h >= heads) h -= heads, ++s;
                if (at[u]) v[u] = *(const uint4 *)at[u];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (at[u]) *(uint4 *)(at[u] + way) = v[u];
        }
    }
}
__global__ void __launch_bounds__(256) kv_grow_copy_kernel(const TableDev t, const PoolDev pool) {
    pdl_wait_prior();
    pdl_launch_dependents();
    const int *const e = t.work + 2 * t.n_seq + 3 * blockIdx.x;
    const int from = e[0];
    if (from >= 0) copy_slots(pool, from, e[1], e[2]);
}
__global__ void __launch_bounds__(256) kv_copy_pages_kernel(const PoolDev pool, const int *src, const int *dst, int n, int *fault) {
    pdl_wait_prior();
    pdl_launch_dependents();
    const int i = blockIdx.x, s = src[i], d = dst[i];
    bool bad = (unsigned)s >= (unsigned)pool.n_pages || (unsigned)d >= (unsigned)pool.n_pages;
    bad |= cta_listed_elsewhere(dst, n, d, i);
    bad |= cta_listed_elsewhere(src, n, d, -1);
    if (bad) {
        if (threadIdx.x == 0) set_fault(fault, ULLM_KV_FAULT_PAGE);
        return;
    }
    copy_slots(pool, s, d, pool.page_size);
}

// ---- plan of a step of trees ----------------------------------------------------------------------------------------
// CTA b < n_seq: the rows of sequence b; the CTAs behind them mark the rows in front of the first sequence and behind the last.  A row walks
// up its ancestors (parents in shared memory), which meet descending indices, so each mask word is complete when the walk leaves it.
constexpr int PLAN_MAX = 4096;
constexpr int PLAN_PAD_CTAS = 4;
__global__ void __launch_bounds__(128) tree_plan_kernel(int n_rows, int n_seq, const int *cu, const int *len, const int *ids, int n_table,
                                                       const int *parent, int *row_seq, int *row_slot, int *row_pos, uint32_t *mask, int words,
                                                       int *fault) {
    __shared__ int par[PLAN_MAX];
    pdl_wait_prior();
    pdl_launch_dependents();
    const int tid = threadIdx.x, b = blockIdx.x;
    bool wild = false; // offsets that decrease or leave the rows: two sequences could own a row, or nobody
    for (int j = tid; n_seq && j <= n_seq; j += 128) wild |= cu[j] < 0 || cu[j] > n_rows || (j < n_seq && cu[j + 1] < cu[j]);
    if (__syncthreads_or(wild)) {
        if (b == 0 && tid == 0) set_fault(fault, ULLM_KV_FAULT_LEN);
        for (int r = b * 128 + tid; r < n_rows; r += gridDim.x * 128) row_seq[r] = -1;
        return;
    }
    if (b >= n_seq) {
        const int first = n_seq ? cu[0] : 0, end = n_seq ? cu[n_seq] : 0, at = (b - n_seq) * 128 + tid;
        for (int r = at; r < first; r += PLAN_PAD_CTAS * 128) row_seq[r] = -1;
        for (int r = end + at; r < n_rows; r += PLAN_PAD_CTAS * 128) row_seq[r] = -1;
        return;
    }
    const int r0 = cu[b], r1 = cu[b + 1];
    const int n = r1 - r0, id = ids ? ids[b] : b;
    int bad = id < 0 || id >= n_table ? ULLM_KV_FAULT_SEQ : 0;
    if (ids && n) { // (entries without rows are padding and may name any row of the table)
        bool twice = false;
        for (int j = tid; j < n_seq; j += 128) twice |= j != b && ids[j] == id && cu[j + 1] != cu[j];
        if (__syncthreads_or(twice)) bad |= ULLM_KV_FAULT_SEQ;
    }
    const int held = bad ? n : len[id], ctx = held - n; // (n is not negative: only a length below it could leave the range)
    if (held < n || (mask && n > 32 * words) || (parent && n > PLAN_MAX)) bad |= ULLM_KV_FAULT_LEN;
    if (bad) {
        if (tid == 0) set_fault(fault, bad);
        for (int i = tid; i < n; i += 128) row_seq[r0 + i] = -1;
        return;
    }
    if (parent) {
        for (int i = tid; i < n; i += 128) {
            int q = parent[r0 + i];
            if (q < -1 || q >= i) {
                set_fault(fault, ULLM_KV_FAULT_PATH);
                q = -1;
            }
            par[i] = q;
        }
        __syncthreads();
    }
    for (int i = tid; i < n; i += 128) {
        uint32_t *const m = mask ? mask + (size_t)(r0 + i) * words : nullptr;
        int depth = 0;
        if (parent) {
            if (m)
                for (int w = i / 32 + 1; w < words; ++w) m[w] = 0;
            int w = i >> 5;
            uint32_t bits = 0;
            for (int q = i; q >= 0; q = par[q], ++depth) {
                while (m && (q >> 5) < w) m[w--] = bits, bits = 0;
                bits |= 1u << (q & 31);
            }
            if (m) {
                m[w] = bits;
                while (--w >= 0) m[w] = 0;
            }
            --depth;
        } else {
            depth = i;
            if (m)
                for (int w = 0; w < words; ++w) m[w] = 32 * w + 31 <= i ? 0xffffffffu : (32 * w > i ? 0u : 0xffffffffu >> (31 - (i & 31)));
        }
        row_seq[r0 + i] = id, row_slot[r0 + i] = ctx + i, row_pos[r0 + i] = ctx + depth;
    }
}

// ---- norm, rotation, cache write ------------------------------------------------------------------------------------
constexpr int ROPE_HPG = 4; // 2: 184 us, 4: 146, 6: 145, 8 with spills: 255 for the long prompt below
struct RopeDev {
    const uint8_t *q, *k, *v;
    long long q_stride, k_stride, v_stride, q_out_stride;
    uint8_t *q_out;
    uint8_t *pk, *pv; // this layer's pages
    long long page_stride, slot_stride, head_stride;
    const float *q_norm, *k_norm, *q_bias, *k_bias, *v_bias;
    const float2 *rope;
    const int *row_seq, *row_slot, *row_pos, *blocks;
    int *fault;
    float eps;
    int n_rows, n_head, n_kv, dim, n_pos, rot, n_table, max_blocks, n_pages, page_size;
};

// Four neighbouring values: as they lie in memory, and as two pairs of f32
template <typename T> struct Io;
template <> struct Io<float> {
    using Raw = float4;
    static __device__ __forceinline__ void widen(const Raw &v, float2 *o) { o[0] = make_float2(v.x, v.y), o[1] = make_float2(v.z, v.w); }
    static __device__ __forceinline__ Raw narrow(const float2 *o) { return make_float4(o[0].x, o[0].y, o[1].x, o[1].y); }
};
template <> struct Io<__half> {
    using Raw = uint2;
    static __device__ __forceinline__ void widen(const Raw &v, float2 *o) { o[0] = __half22float2(*(const __half2 *)&v.x), o[1] = __half22float2(*(const __half2 *)&v.y); }
    static __device__ __forceinline__ Raw narrow(const float2 *o) {
        Raw v;
        *(__half2 *)&v.x = __floats2half2_rn(o[0].x, o[0].y), *(__half2 *)&v.y = __floats2half2_rn(o[1].x, o[1].y);
        return v;
    }
};
template <> struct Io<__nv_bfloat16> {
    using Raw = uint2;
    static __device__ __forceinline__ void widen(const Raw &v, float2 *o) {
        o[0] = make_float2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u)), o[1] = make_float2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
    }
    static __device__ __forceinline__ Raw narrow(const float2 *o) {
        Raw v;
        *(__nv_bfloat162 *)&v.x = __floats2bfloat162_rn(o[0].x, o[0].y), *(__nv_bfloat162 *)&v.y = __floats2bfloat162_rn(o[1].x, o[1].y);
        return v;
    }
};
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { // two products in one instruction
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b));
    return *(float2 *)&r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b), "l"(*(unsigned long long *)&c));
    return *(float2 *)&r;
}
template <typename T> __device__ __forceinline__ typename Io<T>::Raw raw4(const T *p) { return *(const typename Io<T>::Raw *)p; }
template <typename T> __device__ __forceinline__ void put4(T *p, const float2 *o) { *(typename Io<T>::Raw *)p = Io<T>::narrow(o); }

// A group of L lanes (8, 16 or 32: as many as cover head_dim / 8) owns HPG heads of one kind (q, k or v) of one row.  A lane holds eight values of
// a head as two runs of four: with rotate-half one of each half, so that both values of a pair lie in the lane
// (fetched from a neighbour they cost eight shuffles a head), with interleaved pairs and in the part that is not rotated
// neighbouring runs.  Row, page and angles are worked out once for the group's heads.  One pass over the data; for many rows the
// instructions per head count as much as the bytes (16,000 rows of 80 heads of 128 bf16 values, 664 MB: 298 us with eight
// shuffles, a division, scalar arithmetic and addresses for each head; 146 us = 4.5 TB/s as it is, 0.69 of the copy bandwidth).
template <typename X, typename Q, typename KV, int L, int HPG, bool NEOX>
__global__ void __launch_bounds__(256, HPG > 1 ? 4 : 1) qk_norm_rope_kernel(const RopeDev p) {
    pdl_wait_prior();
    pdl_launch_dependents();
    constexpr int GROUPS = 256 / L;
    const int gl = threadIdx.x % L, gq = (p.n_head + HPG - 1) / HPG, gk = (p.n_kv + HPG - 1) / HPG, per_row = gq + 2 * gk;
    const unsigned item = blockIdx.x * (unsigned)GROUPS + threadIdx.x / L;
    const int row = (int)(item / (unsigned)per_row), g = (int)(item % (unsigned)per_row);
    const int kind = g < gq ? 0 : (g < gq + gk ? 1 : 2), head0 = (g - (kind == 0 ? 0 : (kind == 1 ? gq : gq + gk))) * HPG;
    const int heads = min(HPG, (kind == 0 ? p.n_head : p.n_kv) - head0); // of this group
    const unsigned group_lanes = L == 32 ? 0xffffffffu : ((1u << L % 32) - 1u) << (threadIdx.x & 31 & ~(L - 1)); // (a warp's groups may be of different kinds)
    const bool live = row < p.n_rows, mine = live && gl * 8 < p.dim; // lanes behind head_dim only take part in the shuffles
    int seq = -1, slot = 0, pos = 0;
    if (live) seq = p.row_seq[row], slot = p.row_slot[row], pos = p.row_pos[row];
    const bool rotated = gl * 8 < p.rot;
    const int a0 = !NEOX || !rotated ? gl * 8 : gl * 4, b0 = !NEOX || !rotated ? a0 + 4 : p.rot / 2 + gl * 4; // the lane's two runs
    using Raw = typename Io<X>::Raw;
    Raw ra[HPG], rb[HPG];
    {
        const X *src = (const X *)(kind == 0 ? p.q : (kind == 1 ? p.k : p.v)) + row * (kind == 0 ? p.q_stride : (kind == 1 ? p.k_stride : p.v_stride)) + head0 * p.dim;
#pragma unroll
        for (int u = 0; u < HPG; ++u) {
            ra[u] = rb[u] = Raw();
            if (mine && u < heads) ra[u] = raw4(src + u * p.dim + a0), rb[u] = raw4(src + u * p.dim + b0);
        }
    }
    // where the row goes; a row with a position or page outside is left out as a whole
    int page = 0, at = 0;
    if (seq >= 0) {
        const bool ok = seq < p.n_table && slot >= 0 && slot < (long long)p.max_blocks * p.page_size;
        if (ok) {
            const int block = slot / p.page_size;
            page = p.blocks[(size_t)seq * p.max_blocks + block], at = slot - block * p.page_size;
        }
        int bad = !ok ? ULLM_KV_FAULT_LEN : ((unsigned)page >= (unsigned)p.n_pages ? ULLM_KV_FAULT_PAGE : 0);
        if ((unsigned)pos >= (unsigned)p.n_pos) bad |= ULLM_KV_FAULT_POS;
        if (bad) {
            if (g == 0 && gl == 0) set_fault(p.fault, bad);
            seq = -1;
        }
    }
    const bool write = mine && seq >= 0;
    // the lane's four pairs' angles, as (first two, last two)
    float2 c[2] = {{1.f, 1.f}, {1.f, 1.f}}, sn[2] = {{0.f, 0.f}, {0.f, 0.f}};
    if (kind < 2 && write && rotated) {
        const float4 *const t = (const float4 *)(p.rope + (size_t)pos * (p.rot / 2) + gl * 4);
        const float4 u = t[0], v = t[1];
        c[0] = make_float2(u.x, u.z), sn[0] = make_float2(u.y, u.w), c[1] = make_float2(v.x, v.z), sn[1] = make_float2(v.y, v.w);
    }
    const float *const norm = kind == 0 ? p.q_norm : (kind == 1 ? p.k_norm : nullptr);
    const float *const bias = kind == 0 ? p.q_bias : (kind == 1 ? p.k_bias : p.v_bias);
    float2 w[4] = {};
    if (norm && mine) Io<float>::widen(raw4(norm + a0), w), Io<float>::widen(raw4(norm + b0), w + 2);
    const float share = 1.0f / (float)p.dim;
    Q *const q_dst = (Q *)p.q_out + row * p.q_out_stride + head0 * p.dim;
    KV *const kv_dst = (KV *)(kind == 2 ? p.pv : p.pk) + page * p.page_stride + at * p.slot_stride + head0 * p.head_stride;
#pragma unroll
    for (int u = 0; u < HPG; ++u) {
        float2 x[4];
        Io<X>::widen(ra[u], x), Io<X>::widen(rb[u], x + 2);
        if (bias && mine && u < heads) {
            float2 b[4];
            Io<float>::widen(raw4(bias + (size_t)(head0 + u) * p.dim + a0), b), Io<float>::widen(raw4(bias + (size_t)(head0 + u) * p.dim + b0), b + 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e].x += b[e].x, x[e].y += b[e].y;
        }
        if (norm) {
            float2 sq = mul2(x[0], x[0]);
#pragma unroll
            for (int e = 1; e < 4; ++e) sq = fma2(x[e], x[e], sq);
            float ss = sq.x + sq.y;
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group_lanes, ss, o);
            const float inv = rsqrtf(ss * share + p.eps);
            const float2 inv2 = make_float2(inv, inv);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = mul2(mul2(x[e], inv2), w[e]);
        }
        if (kind < 2 && rotated) {
            if (NEOX) { // x[0..1] and x[2..3] are the pairs' first and second values
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 a = x[e], b = x[2 + e], minus = make_float2(-sn[e].x, -sn[e].y);
                    x[e] = fma2(b, minus, mul2(a, c[e])), x[2 + e] = fma2(b, c[e], mul2(a, sn[e]));
                }
            } else { // each x is a pair
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float ce = e & 1 ? c[e / 2].y : c[e / 2].x, se = e & 1 ? sn[e / 2].y : sn[e / 2].x;
                    x[e] = make_float2(x[e].x * ce - x[e].y * se, x[e].x * se + x[e].y * ce);
                }
            }
        }
        if (!write || u >= heads) continue;
        if (kind == 0) put4(q_dst + u * p.dim + a0, x), put4(q_dst + u * p.dim + b0, x + 2);
        else put4(kv_dst + u * p.head_stride + a0, x), put4(kv_dst + u * p.head_stride + b0, x + 2);
    }
}

template <typename X, typename Q, typename KV>
cudaError_t launch_rope_l(const RopeDev &p, int neox, bool pdl, cudaStream_t st) {
    // Heads per group of lanes: several from where that still leaves waves of CTAs (16,000 rows: 145 us, with one head 290; one row: 2.6 us, with one head 2.0).
    const bool many = p.n_rows >= 256;
    auto go = [&](auto kernel, int l, int hpg) {
        const long long items = (long long)p.n_rows * ((p.n_head + hpg - 1) / hpg + 2 * ((p.n_kv + hpg - 1) / hpg)), per = 256 / l;
        return launch_kernel(kernel, dim3((unsigned)((items + per - 1) / per)), dim3(256), 0, st, pdl, p);
    };
    auto with = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value, H = ROPE_HPG;
        if (neox) return many ? go(qk_norm_rope_kernel<X, Q, KV, L, H, true>, L, H) : go(qk_norm_rope_kernel<X, Q, KV, L, 1, true>, L, 1);
        return many ? go(qk_norm_rope_kernel<X, Q, KV, L, H, false>, L, H) : go(qk_norm_rope_kernel<X, Q, KV, L, 1, false>, L, 1);
    };
    if (p.dim <= 64) return with(std::integral_constant<int, 8>());
    if (p.dim <= 128) return with(std::integral_constant<int, 16>());
    return with(std::integral_constant<int, 32>());
}
// queries leave as the pages' type (for the tensor-core attention) or as f32
template <typename X>
cudaError_t launch_rope_x(int q_dtype, int kv_dtype, const RopeDev &p, int neox, bool pdl, cudaStream_t st) {
    const bool q32 = q_dtype == ULLM_DTYPE_F32;
    if (kv_dtype == ULLM_DTYPE_F32) return launch_rope_l<X, float, float>(p, neox, pdl, st);
    if (kv_dtype == ULLM_DTYPE_F16) return q32 ? launch_rope_l<X, float, __half>(p, neox, pdl, st) : launch_rope_l<X, __half, __half>(p, neox, pdl, st);
    return q32 ? launch_rope_l<X, float, __nv_bfloat16>(p, neox, pdl, st) : launch_rope_l<X, __nv_bfloat16, __nv_bfloat16>(p, neox, pdl, st);
}

bool float_dtype(int d) { return d == ULLM_DTYPE_F32 || d == ULLM_DTYPE_F16 || d == ULLM_DTYPE_BF16; }

// Checks shared by the table calls; the pool is filled where the call has one.
int table_check(ullm_cuda_ctx *c, const ullm_kv_pages *kv, const ullm_kv_table *t, size_t n, PoolDev *pool, TableDev *out) {
    if (!kv || !t || !kv->d_k || !kv->d_v || !t->d_blocks || !t->d_len || !t->d_refs || !t->d_fault || !t->d_work)
        return ctx_fail(c, ULLM_ERR_INVALID, "null pointer in a page table call");
    if (const char *m = pool_check(kv, pool)) return ctx_fail(c, ULLM_ERR_FORMAT, "%s", m);
    if (!t->n_seq || !t->max_blocks || t->n_seq > INT32_MAX / 16) return ctx_fail(c, ULLM_ERR_FORMAT, "a table has at least one row and one block");
    if (t->max_blocks > (size_t)(INT32_MAX / 2) / kv->page_size) return ctx_fail(c, ULLM_ERR_FORMAT, "a sequence would pass 2^30 tokens");
    if (n > t->n_seq) return ctx_fail(c, ULLM_ERR_FORMAT, "%zu entries for a table of %zu rows", n, t->n_seq);
    if (t->work_bytes < ullm_cuda_kv_work_bytes(kv->n_pages, t->n_seq))
        return ctx_fail(c, ULLM_ERR_FORMAT, "the table's work area has %zu bytes, %zu are needed", t->work_bytes, ullm_cuda_kv_work_bytes(kv->n_pages, t->n_seq));
    if ((uintptr_t)t->d_work % 4 || (uintptr_t)t->d_blocks % 4 || (uintptr_t)t->d_len % 4 || (uintptr_t)t->d_refs % 4 || (uintptr_t)t->d_fault % 4)
        return ctx_fail(c, ULLM_ERR_FORMAT, "table arrays must be 4-byte aligned");
    out->blocks = t->d_blocks, out->len = t->d_len, out->refs = t->d_refs, out->fault = t->d_fault;
    out->n_seq = (int)t->n_seq, out->max_blocks = (int)t->max_blocks, out->work = (int *)t->d_work;
    return ULLM_OK;
}

// CTAs per entry for work on all matrices of a pool, so that about twelve CTAs of 128 threads fall on an SM
unsigned mats_per_wave(const ullm_cuda_ctx *c, const PoolDev &pool, size_t n) {
    const size_t mats = (size_t)pool.n_layer * 2, all = 12 * (size_t)c->dev.sm_count;
    return (unsigned)std::min(mats, std::max((size_t)1, all / n));
}

} // namespace
} // namespace ullm

using namespace ullm;

size_t ullm_cuda_kv_work_bytes(size_t n_pages, size_t n_seq) { return grow_work_ints(n_pages, n_seq) * 4; }

int ullm_cuda_kv_fork_dev(ullm_cuda_ctx *c, const ullm_kv_pages *kv, const ullm_kv_table *t, const int32_t *d_src, const int32_t *d_dst, size_t n,
                          void *stream) {
    if (!c || (n && (!d_src || !d_dst))) return ULLM_ERR_INVALID;
    PoolDev pool;
    TableDev td;
    if (int rc = table_check(c, kv, t, n, &pool, &td)) return rc;
    if (!ints_aligned(d_src, d_dst)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    if (!n) return ULLM_OK;
    DeviceGuard guard(c->device);
    ULLM_CUDA_TRY(c, launch_kernel(kv_fork_kernel, dim3((unsigned)n), dim3(128), 0, stream ? (cudaStream_t)stream : c->stream, c->use_pdl, td, pool.page_size,
                                   pool.n_pages, d_src, d_dst, (int)n));
    return ULLM_OK;
}

int ullm_cuda_kv_grow_dev(ullm_cuda_ctx *c, const ullm_kv_pages *kv, const ullm_kv_table *t, const int32_t *d_seq, const int32_t *d_add, size_t n,
                          void *stream) {
    if (!c || (n && (!d_seq || !d_add))) return ULLM_ERR_INVALID;
    PoolDev pool;
    TableDev td;
    if (int rc = table_check(c, kv, t, n, &pool, &td)) return rc;
    if (!ints_aligned(d_seq, d_add)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    if (!n) return ULLM_OK;
    DeviceGuard guard(c->device);
    const cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    ULLM_CUDA_TRY(c, launch_kernel(kv_grow_plan_kernel, dim3(1), dim3(1024), 0, st, c->use_pdl, td, pool.page_size, pool.n_pages, d_seq, d_add, (int)n));
    ULLM_CUDA_TRY(c, launch_kernel(kv_grow_copy_kernel, dim3((unsigned)n, mats_per_wave(c, pool, n)), dim3(256), 0, st, c->use_pdl, td, pool));
    return ULLM_OK;
}

int ullm_cuda_kv_accept_dev(ullm_cuda_ctx *c, const ullm_kv_pages *kv, const ullm_kv_table *t, const int32_t *d_seq, const int32_t *d_draft,
                            const int32_t *d_path, const int32_t *d_kept, size_t n, size_t max_path, void *stream) {
    if (!c || (n && (!d_seq || !d_draft || !d_path || !d_kept))) return ULLM_ERR_INVALID;
    PoolDev pool;
    TableDev td;
    if (int rc = table_check(c, kv, t, n, &pool, &td)) return rc;
    if (!ints_aligned(d_seq, d_draft, d_path, d_kept)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    if (max_path > INT32_MAX / 2) return ctx_fail(c, ULLM_ERR_FORMAT, "max_path is too large");
    if (!n) return ULLM_OK;
    DeviceGuard guard(c->device);
    const cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    ULLM_CUDA_TRY(c, launch_kernel(kv_accept_move_kernel, dim3((unsigned)n, mats_per_wave(c, pool, n)), dim3(128), 0, st, c->use_pdl, td, pool, d_seq, d_draft,
                                   d_path, d_kept, (int)n, (int)max_path));
    ULLM_CUDA_TRY(c, launch_kernel(kv_accept_end_kernel, dim3((unsigned)n), dim3(128), 0, st, c->use_pdl, td, pool.page_size, pool.n_pages, d_seq, d_draft, d_kept));
    return ULLM_OK;
}

int ullm_cuda_kv_trim_dev(ullm_cuda_ctx *c, const ullm_kv_pages *kv, const ullm_kv_table *t, const int32_t *d_seq, const int32_t *d_new_len, size_t n,
                          void *stream) {
    if (!c || (n && !d_seq)) return ULLM_ERR_INVALID;
    PoolDev pool;
    TableDev td;
    if (int rc = table_check(c, kv, t, n, &pool, &td)) return rc;
    if (!ints_aligned(d_seq, d_new_len)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    if (!n) return ULLM_OK;
    DeviceGuard guard(c->device);
    ULLM_CUDA_TRY(c, launch_kernel(kv_trim_kernel, dim3((unsigned)n), dim3(128), 0, stream ? (cudaStream_t)stream : c->stream, c->use_pdl, td, pool.page_size,
                                   pool.n_pages, d_seq, d_new_len, (int)n));
    return ULLM_OK;
}

int ullm_cuda_kv_copy_pages_dev(ullm_cuda_ctx *c, const ullm_kv_pages *kv, const int32_t *d_src, const int32_t *d_dst, size_t n, int32_t *d_fault,
                                void *stream) {
    if (!c || !kv || !kv->d_k || !kv->d_v || (n && (!d_src || !d_dst))) return ULLM_ERR_INVALID;
    PoolDev pool;
    if (const char *m = pool_check(kv, &pool)) return ctx_fail(c, ULLM_ERR_FORMAT, "%s", m);
    if (!ints_aligned(d_src, d_dst, d_fault)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    if (n > kv->n_pages) return ctx_fail(c, ULLM_ERR_FORMAT, "%zu copies in a pool of %zu pages", n, kv->n_pages);
    if (!n) return ULLM_OK;
    DeviceGuard guard(c->device);
    ULLM_CUDA_TRY(c, launch_kernel(kv_copy_pages_kernel, dim3((unsigned)n, mats_per_wave(c, pool, n)), dim3(256), 0, stream ? (cudaStream_t)stream : c->stream,
                                   c->use_pdl, pool, d_src, d_dst, (int)n, d_fault));
    return ULLM_OK;
}

int ullm_cuda_tree_plan_dev(ullm_cuda_ctx *c, size_t n_rows, size_t n_seq, const int32_t *d_cu, const int32_t *d_len, const int32_t *d_ids, size_t n_table,
                            const int32_t *d_parent, int32_t *d_row_seq, int32_t *d_row_slot, int32_t *d_row_pos, uint32_t *d_mask, size_t mask_words,
                            int32_t *d_fault, void *stream) {
    if (!c || (n_seq && (!d_cu || !d_len)) || (n_rows && (!d_row_seq || !d_row_slot || !d_row_pos))) return ULLM_ERR_INVALID;
    if (n_rows > INT32_MAX / 2 || n_seq > INT32_MAX / 2 || n_table > INT32_MAX / 2) return ctx_fail(c, ULLM_ERR_FORMAT, "too many rows or sequences");
    if (d_mask && (mask_words == 0 || mask_words > 65536)) return ctx_fail(c, ULLM_ERR_FORMAT, "a mask has 1 to 65536 words per row");
    if (!ints_aligned(d_cu, d_len, d_ids, d_parent, d_row_seq, d_row_slot, d_row_pos, d_mask, d_fault)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    if (!n_rows) return ULLM_OK;
    DeviceGuard guard(c->device);
    ULLM_CUDA_TRY(c, launch_kernel(tree_plan_kernel, dim3((unsigned)(n_seq + PLAN_PAD_CTAS)), dim3(128), 0, stream ? (cudaStream_t)stream : c->stream, c->use_pdl,
                                   (int)n_rows, (int)n_seq, d_cu, d_len, d_ids, (int)n_table, d_parent, d_row_seq, d_row_slot, d_row_pos, d_mask,
                                   (int)mask_words, d_fault));
    return ULLM_OK;
}

int ullm_cuda_qk_norm_rope_dev(ullm_cuda_ctx *c, const ullm_qk_norm_rope *a, void *stream) {
    if (!c || !a || !a->kv) return ULLM_ERR_INVALID;
    if (a->n_rows && (!a->kv->d_k || !a->kv->d_v || !a->d_q || !a->d_k || !a->d_v || !a->d_q_out || !a->d_rope || !a->d_row_seq || !a->d_row_slot || !a->d_row_pos ||
                      !a->d_blocks))
        return ctx_fail(c, ULLM_ERR_INVALID, "null pointer in a norm and rotation call");
    PoolDev pool;
    if (const char *m = pool_check(a->kv, &pool)) return ctx_fail(c, ULLM_ERR_FORMAT, "%s", m);
    if (!float_dtype(a->x_dtype) || !float_dtype(a->q_dtype)) return ctx_fail(c, ULLM_ERR_UNSUPPORTED, "projections and queries are f32, f16 or bf16");
    if (a->q_dtype != ULLM_DTYPE_F32 && a->q_dtype != a->kv->dtype) return ctx_fail(c, ULLM_ERR_UNSUPPORTED, "queries leave as f32 or as the pages' type");
    if (a->layer >= a->kv->n_layer) return ctx_fail(c, ULLM_ERR_FORMAT, "layer %zu of a pool of %zu", a->layer, a->kv->n_layer);
    if (!a->n_head || a->n_head > 65535 || a->n_rows > INT32_MAX / 2) return ctx_fail(c, ULLM_ERR_FORMAT, "bad head or row count");
    const size_t dim = a->kv->head_dim, rot = a->rot_dim ? a->rot_dim : dim;
    if (rot % 16 || rot > dim) return ctx_fail(c, ULLM_ERR_FORMAT, "rot_dim must be a multiple of 16, at most head_dim");
    if (!a->d_q_norm != !a->d_k_norm) return ctx_fail(c, ULLM_ERR_FORMAT, "norm weights for both queries and keys, or for neither");
    if (!a->n_pos || a->n_pos > INT32_MAX || !a->n_table || a->n_table > INT32_MAX / 2 || !a->max_blocks || a->max_blocks > (size_t)(INT32_MAX / 2) / a->kv->page_size)
        return ctx_fail(c, ULLM_ERR_FORMAT, "bad size of the rotation table or of the page table");
    const size_t xb = dtype_bytes(a->x_dtype), qb = dtype_bytes(a->q_dtype), qd = a->n_head * dim, kvd = a->kv->n_kv_head * dim;
    const size_t qs = a->q_stride ? a->q_stride : qd, ks = a->k_stride ? a->k_stride : kvd, vs = a->v_stride ? a->v_stride : kvd;
    const size_t os = a->q_out_stride ? a->q_out_stride : qd;
    if (qs < qd || ks < kvd || vs < kvd || os < qd) return ctx_fail(c, ULLM_ERR_FORMAT, "row strides must cover all heads");
    if (qs * xb % 16 || ks * xb % 16 || vs * xb % 16 || os * qb % 16 || (uintptr_t)a->d_q % 16 || (uintptr_t)a->d_k % 16 || (uintptr_t)a->d_v % 16 ||
        (uintptr_t)a->d_q_out % 16)
        return ctx_fail(c, ULLM_ERR_FORMAT, "rows must start on 16-byte boundaries");
    const void *aligned[6] = {a->d_q_norm, a->d_k_norm, a->d_q_bias, a->d_k_bias, a->d_v_bias, a->d_rope};
    for (const void *p : aligned)
        if ((uintptr_t)p % 16) return ctx_fail(c, ULLM_ERR_FORMAT, "norm weights, biases and the rotation table must be 16-byte aligned");
    if (!ints_aligned(a->d_row_seq, a->d_row_slot, a->d_row_pos, a->d_blocks, a->d_fault)) return ctx_fail(c, ULLM_ERR_FORMAT, "lists must be 4-byte aligned");
    const size_t items = a->n_rows * (a->n_head + 2 * a->kv->n_kv_head);
    if (items >= (size_t)INT32_MAX) return ctx_fail(c, ULLM_ERR_FORMAT, "too many rows for one call");
    if (!a->n_rows) return ULLM_OK;
    RopeDev p;
    p.q = (const uint8_t *)a->d_q, p.k = (const uint8_t *)a->d_k, p.v = (const uint8_t *)a->d_v, p.q_out = (uint8_t *)a->d_q_out;
    p.q_stride = (long long)qs, p.k_stride = (long long)ks, p.v_stride = (long long)vs, p.q_out_stride = (long long)os;
    p.pk = pool.k + (long long)a->layer * pool.layer_stride * pool.elem_bytes, p.pv = pool.v + (long long)a->layer * pool.layer_stride * pool.elem_bytes;
    p.page_stride = pool.page_stride, p.slot_stride = pool.slot_stride, p.head_stride = pool.head_stride;
    p.q_norm = a->d_q_norm, p.k_norm = a->d_k_norm, p.q_bias = a->d_q_bias, p.k_bias = a->d_k_bias, p.v_bias = a->d_v_bias;
    p.rope = (const float2 *)a->d_rope, p.row_seq = a->d_row_seq, p.row_slot = a->d_row_slot, p.row_pos = a->d_row_pos, p.blocks = a->d_blocks;
    p.fault = a->d_fault, p.eps = a->eps, p.n_rows = (int)a->n_rows, p.n_head = (int)a->n_head, p.n_kv = pool.n_kv_head, p.dim = pool.head_dim;
    p.n_pos = (int)a->n_pos, p.rot = (int)rot, p.n_table = (int)a->n_table, p.max_blocks = (int)a->max_blocks, p.n_pages = pool.n_pages, p.page_size = pool.page_size;
    DeviceGuard guard(c->device);
    const cudaStream_t st = stream ? (cudaStream_t)stream : c->stream;
    cudaError_t e;
    if (a->x_dtype == ULLM_DTYPE_F32) e = launch_rope_x<float>(a->q_dtype, a->kv->dtype, p, a->neox != 0, c->use_pdl, st);
    else if (a->x_dtype == ULLM_DTYPE_F16) e = launch_rope_x<__half>(a->q_dtype, a->kv->dtype, p, a->neox != 0, c->use_pdl, st);
    else e = launch_rope_x<__nv_bfloat16>(a->q_dtype, a->kv->dtype, p, a->neox != 0, c->use_pdl, st);
    ULLM_CUDA_TRY(c, e);
    return ULLM_OK;
}
