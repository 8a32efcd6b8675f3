"""What the operators over a paged cache have to give, one entry after the other and in 64 bits: the rules of
include/ullm_cuda.h written as plain Python, apart from the kernels."""
import math

import numpy as np

NO_PAGES, SEQ, LEN, PAGE, PATH, SHARED, POS = (1 << i for i in range(7))


class Tables:
    """Tables and pools [layer, page, slot, head, dim] (k, v: anything that can be indexed and assigned)."""

    def __init__(self, n_seq, max_blocks, n_pages, page_size, k, v):
        self.blocks = np.full((n_seq, max_blocks), -7, np.int64)
        self.len = np.zeros(n_seq, np.int64)
        self.refs = np.zeros(n_pages, np.int64)
        self.fault, self.ps, self.k, self.v = 0, page_size, k, v

    def held(self, s):
        return -(-int(self.len[s]) // self.ps)

    def ok_seq(self, s, listed):
        return 0 <= s < len(self.len) and list(listed).count(s) == 1

    def fork(self, src, dst):
        before = self.len.copy()
        for s, d in zip(src, dst):
            if not (0 <= s < len(before) and 0 <= d < len(before)) or s == d or list(dst).count(d) > 1 or d in list(src) or before[d] != 0:
                self.fault |= SEQ
                continue
            n = -(-int(before[s]) // self.ps)
            if before[s] < 0 or n > self.blocks.shape[1]:
                self.fault |= LEN
                continue
            pages = self.blocks[s, :n]
            if ((pages < 0) | (pages >= len(self.refs))).any():
                self.fault |= PAGE
                continue
            self.blocks[d, :n] = pages
            self.len[d] = before[s]
            for p in pages:
                self.refs[p] += 1

    def grow(self, seq, add):
        refs, plan, total = self.refs.copy(), [], 0
        for s, a in zip(seq, add):
            if not self.ok_seq(s, seq):
                self.fault |= SEQ
                continue
            n = int(self.len[s])
            if n < 0 or a < 0 or n + a > self.blocks.shape[1] * self.ps:
                self.fault |= LEN
                continue
            copy = False
            if a > 0 and n % self.ps:
                last = self.blocks[s, n // self.ps]
                if not 0 <= last < len(refs):
                    self.fault |= PAGE
                    continue
                copy = refs[last] > 1
            have, want = -(-n // self.ps), -(-(n + a) // self.ps)
            plan.append((s, a, n, copy, have, want))
            total += want - have + copy
        free = [p for p in range(len(refs)) if refs[p] == 0]
        if total > len(free):
            self.fault |= NO_PAGES
            return
        for s, a, n, copy, have, want in plan:
            if copy:
                old, new = int(self.blocks[s, have - 1]), free.pop(0)
                self.k[:, new, :n % self.ps] = self.k[:, old, :n % self.ps]
                self.v[:, new, :n % self.ps] = self.v[:, old, :n % self.ps]
                self.refs[old] -= 1
                self.refs[new] = 1
                self.blocks[s, have - 1] = new
            for b in range(have, want):
                self.blocks[s, b] = free.pop(0)
                self.refs[self.blocks[s, b]] = 1
            self.len[s] = n + a

    def release(self, s, keep, have):
        for b in range(keep, have):
            p = self.blocks[s, b]
            if not 0 <= p < len(self.refs) or self.refs[p] <= 0:
                self.fault |= PAGE
            else:
                self.refs[p] -= 1

    def accept(self, seq, draft, path, kept):
        refs, done = self.refs.copy(), []
        for i, s in enumerate(seq):
            if not self.ok_seq(s, seq):
                self.fault |= SEQ
                continue
            n, nd, nk = int(self.len[s]), int(draft[i]), int(kept[i])
            if nd < 0 or nd > n or nk < 0 or nk > nd or nk > path.shape[1] or self.held(s) > self.blocks.shape[1]:
                self.fault |= LEN
                continue
            p, base, bad = [int(x) for x in path[i, :nk]], n - nd, 0
            where = lambda t: (int(self.blocks[s, t // self.ps]), t % self.ps)  # noqa: E731
            for j, x in enumerate(p):
                if not 0 <= x < nd or (j and x <= p[j - 1]):
                    bad |= PATH
                elif x != j:
                    a, b = where(base + x)[0], where(base + j)[0]
                    if not (0 <= a < len(refs) and 0 <= b < len(refs)):
                        bad |= PAGE
                    elif refs[b] != 1:
                        bad |= SHARED
            self.fault |= bad
            if bad:
                continue
            for j, x in enumerate(p):
                if x != j:
                    (a, i0), (b, i1) = where(base + x), where(base + j)
                    self.k[:, b, i1], self.v[:, b, i1] = self.k[:, a, i0].copy(), self.v[:, a, i0].copy()
            done.append((s, base + nk))
        for s, n in done:
            self.release(s, -(-n // self.ps), self.held(s))
            self.len[s] = n

    def trim(self, seq, new=None):
        for i, s in enumerate(seq):
            if not self.ok_seq(s, seq):
                self.fault |= SEQ
                continue
            want = 0 if new is None else int(new[i])
            if want < 0 or want > self.len[s] or self.held(s) > self.blocks.shape[1]:
                self.fault |= LEN
                continue
            self.release(s, -(-want // self.ps), self.held(s))
            self.len[s] = want


def plan(cu, lens, parents, n_rows, words=None, ids=None):
    """(row_seq, row_slot, row_pos, mask, fault); rows that are not written hold None / -9."""
    seq, slot, pos = (np.full(n_rows, -9, np.int64) for _ in range(3))
    mask = np.full((n_rows, words or 1), 0xEEEEEEEE, np.uint32)
    fault = 0
    for b in range(len(cu) - 1):
        r0, n = cu[b], cu[b + 1] - cu[b]
        t = b if ids is None else ids[b]
        if not 0 <= t < len(lens):
            fault |= SEQ
            seq[r0:r0 + n] = -1
            continue
        ctx = lens[t] - n
        if ctx < 0 or (words and n > 32 * words):
            fault |= LEN
            seq[r0:r0 + n] = -1
            continue
        for i in range(n):
            chain, q = [i], i - 1 if parents is None else parents[r0 + i]
            if parents is not None and not -1 <= q < i:
                fault |= PATH
                q = -1
            while q >= 0:
                chain.append(q)
                if parents is None:
                    q -= 1
                else:
                    q = parents[r0 + q] if -1 <= parents[r0 + q] < q else -1
            seq[r0 + i], slot[r0 + i], pos[r0 + i] = t, ctx + i, ctx + len(chain) - 1
            if words:
                mask[r0 + i] = 0
                for q in chain:
                    mask[r0 + i, q // 32] |= np.uint32(1 << (q % 32))
    seq[cu[-1]:] = -1
    return seq, slot, pos, mask, fault


def rope_rows(x, heads, norm, eps, cs, rot, neox):
    """Normalised and rotated heads of x [rows, heads * dim] (float64) with cs [rows, rot / 2, 2], and the sum of the
    magnitudes that make up each value."""
    x = np.asarray(x, np.float64)
    t = x.reshape(x.shape[0], heads, -1)
    if norm is not None:
        t = t / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * norm
    out, mag = t.copy(), np.abs(t)
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    out[..., a], out[..., b] = t[..., a] * c - t[..., b] * s, t[..., a] * s + t[..., b] * c
    mag[..., a], mag[..., b] = np.abs(t[..., a] * c) + np.abs(t[..., b] * s), np.abs(t[..., a] * s) + np.abs(t[..., b] * c)
    return out, mag


def attention(q, k, v, see, scale):
    """One sequence: q [n, heads, dim], k and v [keys, kv_heads, dim] in float64, see [n, keys] -> out, sum of p |v| and
    the largest (finite) sum of |q| |k| * scale of each row and head."""
    n, heads, dim = q.shape
    g = heads // k.shape[1]
    out, weight, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, heads))
    for h in range(heads):
        kk, vv = k[:, h // g], v[:, h // g]
        for i in range(n):
            j = np.nonzero(see[i])[0]
            if not len(j):
                continue
            s = kk[j] @ q[i, h] * scale
            with np.errstate(invalid="ignore", over="ignore"):
                p = np.exp(s - s.max())
                p = p / p.sum()
                out[i, h] = (p[:, None] * vv[j]).sum(0)
                weight[i, h] = (p[:, None] * np.abs(vv[j])).sum(0)
            terms = np.abs(kk[j]) @ np.abs(q[i, h])
            size[i, h] = terms[np.isfinite(terms)].max(initial=0) * scale
    return out, weight, size


def tree_parents(n, rng, root=0.1):
    p = np.array([i - 1 - min(int(rng.geometric(0.5)) - 1, i) for i in range(n)], np.int64)
    p[rng.random(n) < root] = -1
    return p


def default_scale(dim):
    return 1.0 / math.sqrt(dim)
