"""GPU tests of the attention over a paged cache against the formula in 64 bits (paged_ref.attention)."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import paged_ref
from test_paged_gpu import DT, ints, make_pool, stream
from ullm_b200 import backend

pytestmark = pytest.mark.gpu


class Case:
    """A step of rows over a pool in which every slot that no sequence uses holds NaN."""

    def __init__(self, ctxs, counts, heads, kv_heads, dim, dtype, ps, layout="slot", q32=False, mask="tree", seed=0, pad=2, layers=2, ids=None, n_table=None,
                 spare=0, extra_words=0, extra_blocks=1, gain=1.5):
        rng = np.random.default_rng(seed)
        self.ps, self.heads, self.kv_heads, self.dim, self.pad = ps, heads, kv_heads, dim, pad
        self.ids = list(range(len(ctxs))) if ids is None else ids
        self.n_table = n_table or len(ctxs)
        self.counts, self.ctxs = counts, ctxs
        self.cu = np.concatenate([[0], np.cumsum(counts)])
        self.rows = int(self.cu[-1])
        need = [-(-(c + n) // ps) for c, n in zip(ctxs, counts)]
        n_pages = sum(need) + 3
        self.max_blocks = max(need) + extra_blocks
        perm = rng.permutation(n_pages)
        self.blocks = np.full((self.n_table, self.max_blocks), -1, np.int64)
        self.lens = np.zeros(self.n_table, np.int64)
        at = 0
        for b, t in enumerate(self.ids):
            self.blocks[t, :need[b]] = perm[at:at + need[b]]
            self.lens[t] = ctxs[b] + counts[b]
            at += need[b]
        self.layer = layers - 1
        self.k, self.v, self.kv = make_pool(layers, n_pages, ps, kv_heads, dim, dtype, layout, seed, spare)
        used = np.zeros((n_pages, ps), bool)
        for t in self.ids:
            tok = np.arange(self.lens[t])
            used[self.blocks[t, tok // ps], tok % ps] = True
        idle = torch.as_tensor(~used).cuda()
        for pool in (self.k, self.v):
            pool[self.layer][idle] = float("nan")
        self.qt = torch.float32 if q32 else DT[dtype][1]
        self.qd = backend.F32 if q32 else DT[dtype][0]
        self.qs, self.os = heads * dim + 16, heads * dim + 8
        g = torch.Generator().manual_seed(seed + 1)
        self.q = (torch.randn(self.rows + pad, self.qs, generator=g) * gain).to(self.qt).cuda()
        self.out = torch.full((self.rows + pad, self.os), 7.0, dtype=self.qt, device="cuda")
        self.words = 0
        self.mask = None
        if mask != "chain":
            self.words = max(1, -(-max(counts) // 32)) + extra_words
            m = np.zeros((self.rows + pad, self.words), np.uint32)
            for b, n in enumerate(counts):
                if mask == "tree":
                    par = paged_ref.tree_parents(n, rng)
                    for i in range(n):
                        if par[i] >= 0:
                            m[self.cu[b] + i] = m[self.cu[b] + par[i]]
                        m[self.cu[b] + i, i // 32] |= np.uint32(1 << (i % 32))
                elif mask == "any":  # also bits of later rows, bits behind the last row, empty rows
                    m[self.cu[b]:self.cu[b] + n] = rng.integers(0, 2 ** 32, (n, self.words), dtype=np.uint64).astype(np.uint32)
                    m[self.cu[b]:self.cu[b] + n][rng.random(n) < 0.3] = 0
            self.mask = m

    def run(self, ctx, op=None, s=None, scale=0.0):
        op = op or backend.TreeAttention(ctx, self.kv, self.heads, dtype=self.qd, scale=scale)
        self.d = [ints(self.cu), ints(self.lens), ints(self.blocks), ints(self.ids), None if self.mask is None else torch.as_tensor(self.mask.view(np.int32)).cuda()]
        op.run_dev(self.layer, self.q.data_ptr(), self.out.data_ptr(), self.rows + self.pad, len(self.ids), self.d[0].data_ptr(), self.d[1].data_ptr(),
                   self.d[2].data_ptr(), self.max_blocks, d_mask=None if self.mask is None else self.d[4].data_ptr(), mask_words=self.words,
                   d_ids=self.d[3].data_ptr(), n_table=self.n_table, q_stride=self.qs, out_stride=self.os, stream=s or stream())
        return op

    def see(self, b):
        n, ctx = self.counts[b], self.ctxs[b]
        s = np.ones((n, ctx + n), bool)
        i = np.arange(n)
        if self.mask is None:
            s[:, ctx:] = i[None] <= i[:, None]
        else:
            m = self.mask[self.cu[b]:self.cu[b] + n]
            s[:, ctx:] = (m[:, i // 32] >> (i % 32).astype(np.uint32)) & 1
        return s

    def check(self, scale=None):
        torch.cuda.synchronize()
        scale = scale or paged_ref.default_scale(self.dim)
        k, v = self.k[self.layer].double().cpu().numpy(), self.v[self.layer].double().cpu().numpy()
        q, out = self.q.double().cpu().numpy(), self.out.double().cpu().numpy()
        half = torch.finfo(self.qt).eps / 2
        worst = 0.0
        for b, t in enumerate(self.ids):
            r0, n, ctx = self.cu[b], self.counts[b], self.ctxs[b]
            tok = np.arange(ctx + n)
            page, at = self.blocks[t, tok // self.ps], tok % self.ps
            qq = q[r0:r0 + n, :self.heads * self.dim].reshape(n, self.heads, self.dim)
            ref, weight, size = paged_ref.attention(qq, k[page, at], v[page, at], self.see(b), scale)
            got = out[r0:r0 + n, :self.heads * self.dim].reshape(ref.shape)
            # 32-bit steps, each half a step of 2^-23: a score of magnitude `size` from dim products, its scale and the distance to the
            # maximum (dim + 4 of `size`, twice for numerator and sum), the power of two (4), sums over the keys and the
            # joining of parts (keys + 64) of the weighted values.  16-bit types: the weights are rounded once (half a step of what
            # they weigh, and of their sum) and the result once (half a step of its value).
            f32 = (2 * (self.dim + 4) * size[..., None] + ctx + n + 72) * 2.0 ** -24 * weight
            bound = f32 + 1e-30
            if self.qt != torch.float32:
                bound = bound + 2 * half * weight + half * (np.abs(ref) + bound) + (2.0 ** -25 if self.qt == torch.float16 else 0.0)
            fine = np.isfinite(ref)
            assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)])
            err = np.abs(np.where(fine, got - np.where(fine, ref, 0), 0))
            worst = max(worst, float((err / np.where(fine, bound, 1)).max(initial=0)))
        assert worst <= 1, worst
        assert bool((self.out[self.rows:] == 7).all()) and bool((self.out[:, self.heads * self.dim:] == 7).all())


TYPES = [("f16", False), ("bf16", False), ("f32", True), ("f16", True), ("bf16", True)]


@pytest.mark.parametrize("dtype,q32", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,ps,layout", [
    (8, 2, 64, 16, "slot"), (8, 1, 128, 32, "head"), (4, 4, 128, 64, "slot"), (6, 2, 64, 8, "head"), (16, 2, 128, 128, "slot"), (2, 2, 64, 256, "slot"),
    (4, 2, 40, 7, "slot"), (3, 3, 256, 1, "head"), (10, 2, 96, 24, "slot"), (4, 1, 8, 16, "head"), (4, 2, 64, 12, "slot"),
])
def test_types_heads_and_pages(ctx, dtype, q32, heads, kv_heads, dim, ps, layout):
    for mask in ("tree", "chain", "any"):
        c = Case([0, 1, 37, 200, 300], [1, 5, 17, 33, 2], heads, kv_heads, dim, dtype, ps, layout, q32, mask, seed=dim + ps, spare=8 if layout == "slot" else 0)
        c.run(ctx)
        c.check()


@pytest.mark.parametrize("dtype,dim", [("f16", 64), ("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("ctx_len,n", [(0, 1), (0, 2), (1, 1), (62, 1), (63, 1), (64, 1), (63, 2), (126, 1), (127, 1), (128, 1), (120, 9), (255, 1), (256, 1), (250, 70),
                                       (1000, 1), (383, 130), (5000, 3)])
def test_lengths_around_the_blocks(ctx, dtype, dim, ctx_len, n):
    for heads, kv_heads in ((4, 1), (2, 2)):
        c = Case([ctx_len], [n], heads, kv_heads, dim, dtype, 16, mask="tree", seed=ctx_len + n, q32=dtype == "f32")
        c.run(ctx)
        c.check()


def test_many_short_sequences_and_table_rows_in_any_order(ctx):
    rng = np.random.default_rng(9)
    counts = [int(x) for x in rng.integers(0, 4, 700)]
    ctxs = [int(x) for x in rng.integers(0, 20, 700)]
    for dtype in ("bf16", "f32"):
        c = Case(ctxs, counts, 4, 2, 64, dtype, 8, mask="tree", ids=[int(x) for x in rng.permutation(900)[:700]], n_table=900, q32=dtype == "f32")
        c.run(ctx)
        c.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_long_chain_is_a_causal_prompt(ctx, dtype):
    c = Case([70, 0], [300, 257], 4, 1, 64, dtype, 16, mask="chain", q32=dtype == "f32")
    c.run(ctx)
    c.check()


@pytest.mark.parametrize("dtype,dim,ps", [("f16", 64, 16), ("bf16", 128, 32), ("bf16", 128, 24), ("f32", 64, 16)])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(ctx, dtype, dim, ps):
    """NaN and infinities in drafted tokens' keys and values (an unverified node may hold anything)."""
    c = Case([130, 0, 40], [40, 9, 33], 4, 2, dim, dtype, ps, mask="any", seed=5, q32=dtype == "f32", gain=0.5)
    rng = np.random.default_rng(6)
    for b, t in enumerate(c.ids):
        for what in (float("nan"), float("inf"), -float("inf")):
            for pool in (c.k, c.v):
                if pool is c.k and not np.isnan(what):
                    continue  # an infinite key gives scores of either sign and NaN with zeros: NaN stands for it
                tok = c.ctxs[b] + int(rng.integers(c.counts[b]))
                pool[c.layer, int(c.blocks[t, tok // ps]), tok % ps, :, ::3] = what
    c.run(ctx)
    c.check()


def test_extreme_scores(ctx):
    """Scores of a few hundred: one key takes all the weight, and the running maximum grows block after block."""
    for dtype in ("bf16", "f32"):
        c = Case([900, 300], [8, 20], 4, 1, 64, dtype, 16, mask="tree", gain=40.0, q32=dtype == "f32")
        ramp = torch.linspace(0.01, 1.0, 1000, device="cuda")
        for t in c.ids:
            tok = np.arange(c.lens[t])
            page, at = torch.as_tensor(c.blocks[t, tok // c.ps]).cuda(), torch.as_tensor(tok % c.ps).cuda()
            c.k[c.layer, page, at] = (c.k[c.layer, page, at].float() * ramp[: len(tok), None, None]).to(c.k.dtype)
        c.run(ctx)
        c.check()


def test_scale_and_pages_outside_the_pool(ctx):
    c = Case([200], [6], 4, 2, 64, "f16", 16, mask="tree")
    c.run(ctx, scale=0.3)
    c.check(scale=0.3)
    # the third and the last page are no pages: their keys and values are zeros
    c.blocks[0, 2], c.blocks[0, 12] = c.kv.n_pages, -4
    for ps_dim in ((16, 64),):
        c.run(ctx)
        torch.cuda.synchronize()
        tok = np.arange(206)
        page = c.blocks[0, tok // 16]
        ok = (page >= 0) & (page < c.kv.n_pages)
        k, v = (np.where(ok[:, None, None], p[c.layer].double().cpu().numpy()[np.where(ok, page, 0), tok % 16], 0) for p in (c.k, c.v))
        q = c.q[:6, :256].double().cpu().numpy().reshape(6, 4, 64)
        ref, weight, _ = paged_ref.attention(q, k, v, c.see(0), paged_ref.default_scale(64))
        err = np.abs(c.out[:6, :256].double().cpu().numpy().reshape(ref.shape) - ref)
        assert (err <= 2.0 ** -11 * (np.abs(ref) + 2 * weight) * 1.02 + 2.0 ** -25).all()


def test_rows_of_inconsistent_sequences_become_zeros(ctx):
    for dtype in ("f16", "f32"):
        c = Case([40, 60, 20, 30], [3, 4, 2, 5], 4, 2, 64, dtype, 16, mask="tree", q32=dtype == "f32")
        c.lens[0], c.lens[1] = 2, c.max_blocks * 16 + 1  # fewer tokens than rows; more than the table holds
        c.ids[2] = 77                                       # no such row
        c.run(ctx)
        torch.cuda.synchronize()
        assert bool((c.out[:9, :256] == 0).all()) and bool((c.out[9:14, :256] != 0).any()) and bool((c.out[14:] == 7).all())


def test_repeated_calls_are_bit_equal_and_streams_and_graphs_work(ctx):
    for dtype, dim in (("bf16", 128), ("f32", 64)):
        c = Case([3000, 10, 700], [9, 64, 1], 8, 2, dim, dtype, 32, mask="tree", q32=dtype == "f32")
        op = c.run(ctx)
        c.check()
        first = c.out.clone()
        keep = c.d
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c.run(ctx, op, s=side.cuda_stream)
        side.synchronize()
        assert torch.equal(c.out, first)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            d = c.d
            op.run_dev(c.layer, c.q.data_ptr(), c.out.data_ptr(), c.rows + c.pad, 3, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), c.max_blocks,
                       d_mask=d[4].data_ptr(), mask_words=c.words, d_ids=d[3].data_ptr(), n_table=3, q_stride=c.qs, out_stride=c.os, stream=side.cuda_stream)
        c.out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, first)
        # the lengths are read when the graph runs: one committed token less in the first sequence, the drafts one slot earlier
        c.ctxs[0] -= 1
        c.lens[0] -= 1
        c.d[1].copy_(ints(c.lens))
        g.replay()
        c.check()
        assert not torch.equal(c.out, first)
        del keep


def test_own_stream_and_two_calls_at_once(ctx):
    """A null stream is the context's own; two objects have work areas of their own and may run at the same time."""
    a = Case([4000, 900], [7, 3], 8, 2, 128, "bf16", 16, mask="tree", seed=1)
    b = Case([2500, 1900], [5, 30], 8, 2, 128, "bf16", 16, mask="tree", seed=2)
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    ops = [None, None]
    for _ in range(5):
        for i, c in enumerate((a, b)):
            c.out.fill_(7)
            torch.cuda.synchronize()
        for i, c in enumerate((a, b)):
            ops[i] = c.run(ctx, ops[i], s=s[i].cuda_stream)
        a.check()
        b.check()
    a.out.fill_(7)
    torch.cuda.synchronize()
    op = backend.TreeAttention(ctx, a.kv, a.heads)
    op.run_dev(a.layer, a.q.data_ptr(), a.out.data_ptr(), a.rows + a.pad, 2, a.d[0].data_ptr(), a.d[1].data_ptr(), a.d[2].data_ptr(), a.max_blocks,
               d_mask=a.d[4].data_ptr(), mask_words=a.words, d_ids=a.d[3].data_ptr(), n_table=2, q_stride=a.qs, out_stride=a.os)
    ctx.synchronize()
    a.check()


def test_offsets_beyond_32_bits(ctx):
    """A pool of more than 4 G elements: the pages used lie behind its first 2^32 values."""
    ps, heads, dim, n_pages = 64, 8, 128, (1 << 32) // (64 * 8 * 128) + 40
    k = torch.zeros((1, n_pages, ps, heads, dim), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator(device="cuda").manual_seed(3)
    for p in (k, v):
        p[0, -30:] = torch.randn((30, ps, heads, dim), generator=g, device="cuda").half()
    kv = backend.KvPages(backend.F16, 1, n_pages, ps, heads, dim, k.data_ptr(), v.data_ptr())
    c = Case([600, 500], [5, 9], 16, 8, dim, "f16", ps, mask="tree", layers=1)
    c.blocks = np.where(c.blocks >= 0, n_pages - 1 - c.blocks, -1)
    c.k, c.v, c.kv = k, v, kv
    c.run(ctx)
    torch.cuda.synchronize()
    lo = n_pages - 30
    c.k, c.v, c.blocks = k[:, lo:], v[:, lo:], np.where(c.blocks >= 0, c.blocks - lo, -1)
    c.check()


def test_a_step_of_speculative_decoding(ctx):
    """The operators as they are used: tables -> plan -> norm, rotation, cache write -> attention -> accept, over two layers and
    three rounds with a forked sequence; each step's attention sees what the steps before kept."""
    layers, ps, heads, kv_heads, dim, n_seq, max_blocks, n_pages = 2, 16, 8, 2, 64, 4, 12, 40
    rng = np.random.default_rng(21)
    k, v, kv = make_pool(layers, n_pages, ps, kv_heads, dim, "f32", "slot", 8)
    blocks, lens, refs, fault = ints(np.full((n_seq, max_blocks), -1)), ints(np.zeros(n_seq)), ints(np.zeros(n_pages)), ints([0])
    t = backend.KvTable(ctx, kv, blocks.data_ptr(), lens.data_ptr(), refs.data_ptr(), fault.data_ptr(), n_seq, max_blocks)
    cs = np.stack([np.cos(a := np.arange(200)[:, None] * 1e4 ** (-np.arange(dim // 2) / (dim // 2))), np.sin(a)], -1).astype(np.float32)
    d_cs, w = torch.as_tensor(cs).cuda(), [1 + 0.1 * rng.standard_normal(dim).astype(np.float32) for _ in range(2)]
    d_w = [torch.as_tensor(x).cuda() for x in w]
    rope = backend.QkNormRope(ctx, kv, heads, backend.F32, d_cs.data_ptr(), 200, neox=True, d_q_norm=d_w[0].data_ptr(), d_k_norm=d_w[1].data_ptr(), eps=1e-6)
    attn = backend.TreeAttention(ctx, kv, heads)
    history = {0: [[] for _ in range(layers)], 1: [[] for _ in range(layers)]}  # kept (key, value) rows of each sequence and layer
    active, st = [0], stream()
    for rnd in range(4):
        if rnd == 2:
            d_src, d_dst = ints([0]), ints([1])
            t.fork_dev(d_src.data_ptr(), d_dst.data_ptr(), 1, stream=st)
            history[1] = [list(x) for x in history[0]]
            active = [0, 1]
        counts = [int(rng.integers(30, 40)) if rnd == 0 else int(rng.integers(3, 20)) for _ in active]
        ids, add = ints(active), ints(counts)
        t.grow_dev(ids.data_ptr(), add.data_ptr(), len(active), stream=st)
        parents = [np.arange(n) - 1 if rnd == 0 else paged_ref.tree_parents(n, rng) for n in counts]
        cu = np.concatenate([[0], np.cumsum(counts)])
        rows, words = int(cu[-1]), 2
        d_cu, d_par = ints(cu), ints(np.concatenate(parents))
        seq, slot, pos = (ints(np.zeros(rows)) for _ in range(3))
        mask = torch.zeros((rows, words), dtype=torch.int32, device="cuda")
        ctx.tree_plan_dev(rows, len(active), d_cu.data_ptr(), lens.data_ptr(), d_par.data_ptr(), seq.data_ptr(), slot.data_ptr(), pos.data_ptr(), mask.data_ptr(), words,
                          fault.data_ptr(), ids.data_ptr(), n_seq, st)
        new = {}
        for layer in range(layers):
            x = torch.randn(rows, (heads + 2 * kv_heads) * dim, generator=torch.Generator().manual_seed(100 * rnd + layer)).cuda()
            q, out = torch.empty(rows, heads * dim, device="cuda"), torch.empty(rows, heads * dim, device="cuda")
            p = x.data_ptr()
            rope.run_dev(layer, p, p + heads * dim * 4, p + (heads + kv_heads) * dim * 4, q.data_ptr(), rows, pos.data_ptr(), seq.data_ptr(), slot.data_ptr(), blocks.data_ptr(),
                         n_seq, max_blocks, x_stride=x.shape[1], d_fault=fault.data_ptr(), stream=st)
            attn.run_dev(layer, q.data_ptr(), out.data_ptr(), rows, len(active), d_cu.data_ptr(), lens.data_ptr(), blocks.data_ptr(), max_blocks, d_mask=mask.data_ptr(),
                         mask_words=words, d_ids=ids.data_ptr(), n_table=n_seq, stream=st)
            torch.cuda.synchronize()
            xx = x.double().cpu().numpy()
            for b, s in enumerate(active):
                n, ctx_len = counts[b], len(history[s][layer])
                depth = np.zeros(n, int)
                see = np.zeros((n, ctx_len + n), bool)
                see[:, :ctx_len] = True
                for i in range(n):
                    if parents[b][i] >= 0:
                        see[i], depth[i] = see[parents[b][i]], depth[parents[b][i]] + 1
                    see[i, ctx_len + i] = True
                r = slice(cu[b], cu[b + 1])
                c = cs.astype(np.float64)[ctx_len + depth]
                qq, _ = paged_ref.rope_rows(xx[r, :heads * dim], heads, w[0], 1e-6, c, dim, True)
                kk, _ = paged_ref.rope_rows(xx[r, heads * dim:(heads + kv_heads) * dim], kv_heads, w[1], 1e-6, c, dim, True)
                vv = xx[r, (heads + kv_heads) * dim:].reshape(n, kv_heads, dim)
                new[s, layer] = list(zip(kk, vv))
                both = history[s][layer] + new[s, layer]
                ref, weight, size = paged_ref.attention(qq, np.stack([a for a, _ in both]), np.stack([a for _, a in both]), see, paged_ref.default_scale(dim))
                err = np.abs(out[r].double().cpu().numpy().reshape(ref.shape) - ref)
                # attention's bound (above) and the rotated queries' and keys': (16 + dim / 16) half steps each on scores of magnitude `size`, twice
                bound = (2 * (dim + 4 + 2 * (16 + dim / 16)) * size[..., None] + len(both) + 72) * 2.0 ** -24 * weight
                assert (err <= bound).all(), (rnd, layer, s, float((err / bound).max()))
        path, kept = np.zeros((len(active), 40), int), []
        for b, s in enumerate(active):
            chain, i = [], int(rng.integers(counts[b]))
            while i >= 0:
                chain.insert(0, i)
                i = int(parents[b][i])
            path[b, :len(chain)] = chain
            kept.append(len(chain))
            for layer in range(layers):
                history[s][layer] += [new[s, layer][j] for j in chain]
        d_path, d_kept = ints(path), ints(kept)
        t.accept_dev(ids.data_ptr(), add.data_ptr(), d_path.data_ptr(), d_kept.data_ptr(), len(active), 40, stream=st)
        torch.cuda.synchronize()
        assert int(fault[0]) == 0
        for s in active:
            n = len(history[s][0])
            assert int(lens[s]) == n
            tok = np.arange(n)
            page = blocks[s].cpu().numpy()[tok // ps]
            for layer in range(layers):
                got = v[layer].double().cpu().numpy()[page, tok % ps]
                assert np.array_equal(got, np.stack([a for _, a in history[s][layer]]))
    ids = ints([0, 1])
    t.trim_dev(ids.data_ptr(), None, 2, stream=st)
    torch.cuda.synchronize()
    assert int(refs.abs().sum()) == 0 and int(fault[0]) == 0


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f32", 128), ("f16", 128), ("bf16", 64), ("f32", 96)])
@pytest.mark.parametrize("ctx_len,n", [(0, 1), (7, 1), (8, 1), (63, 1), (64, 1), (61, 6), (130, 40), (1000, 1), (700, 33), (4000, 9)])
def test_32_bit_queries_around_the_blocks(ctx, dtype, dim, ctx_len, n):
    """One row to many over pages of every type: tiles of 16 and of 32 rows (the table's size decides for few rows), whole units and units in many parts."""
    for heads, kv_heads, blocks in ((8, 2, 1), (3, 3, 3000)):
        c = Case([ctx_len, 5], [n, 2], heads, kv_heads, dim, dtype, 16, mask="any", seed=ctx_len + n + dim, q32=True, extra_blocks=blocks)
        c.run(ctx)
        c.check()


@pytest.mark.parametrize("dtype,q32,dim", [("f32", True, 64), ("f16", True, 128), ("bf16", True, 64), ("bf16", False, 128), ("f16", False, 40), ("f32", True, 40)])
def test_infinite_keys_and_values_of_the_context(ctx, dtype, q32, dim):
    """A key whose score is -inf has no weight, one whose score is +inf or NaN makes its rows NaN; an infinite value that a row sees makes it infinite."""
    c = Case([300, 90], [5, 3], 4, 2, dim, dtype, 16, mask="tree", seed=4, q32=q32)
    c.q[:, :4 * dim] = c.q[:, :4 * dim].abs()
    at = lambda b, tok: (c.layer, int(c.blocks[b, tok // 16]), tok % 16)
    c.k[at(0, 17)][:, 3] = -float("inf")
    c.k[at(0, 250)][:, dim - 1] = -float("inf")
    c.v[at(0, 100)][0, 5] = float("inf")
    c.v[at(0, 200)][1, 6] = -float("inf")
    c.k[at(1, 40)][1, 2] = float("inf")
    c.run(ctx)
    c.check()


def test_the_largest_32_bit_values(ctx):
    """Keys, values and queries at the end of the range stay what they are: products of them are finite where the formula's are."""
    big = torch.finfo(torch.float32).max
    for dim in (64, 128, 40):
        c = Case([100], [4], 2, 1, dim, "f32", 16, mask="tree", seed=dim)
        c.q[:, :2 * dim] *= 0.01
        c.q[1, 3], c.q[2, dim + 4] = big, -big
        for tok in range(104):
            page, slot = int(c.blocks[0, tok // 16]), tok % 16
            c.k[c.layer, page, slot, 0, 3:5] = 0
            c.k[c.layer, page, slot, 0, 4] = 1e-38 if tok % 2 else 0
            c.v[c.layer, page, slot, 0, 7] = big if tok == 50 else 0  # (a sum of several would pass the range before it is divided)
        c.run(ctx)
        c.check()


def test_a_work_area_needs_no_preparation(ctx):
    """Whatever the work area held, and whichever calls used it before, a call's result is the same bit by bit."""
    for dtype, dim in (("f32", 64), ("f16", 128), ("f32", 80)):
        c = Case([2500, 300, 0], [7, 40, 1], 8, 2, dim, dtype, 16, mask="tree", q32=dtype == "f32", seed=3)
        op = c.run(ctx)
        c.check()
        first = c.out.clone()
        work = torch.empty(op._a.work_bytes // 4 + 1, dtype=torch.int32, device="cuda")
        op._a.d_work = work.data_ptr()
        for fill in (0, -1, 1, 0x7FC00000):
            work.fill_(fill)
            for _ in range(2):
                c.out.fill_(7)
                c.run(ctx, op)
                torch.cuda.synchronize()
                assert torch.equal(c.out, first)


@pytest.mark.parametrize("dtype,ps", [("f16", 384), ("bf16", 512), ("f16", 128), ("f32", 512)])
def test_sequences_without_keys_beside_large_pages(ctx, dtype, ps):
    """Rows of a sequence whose length is inconsistent see nothing and read no page; the table's last row is one of them."""
    c = Case([40, 700, 0], [3, 9, 2], 4, 2, 64, dtype, ps, mask="tree", q32=dtype == "f32", extra_blocks=0)
    c.lens[0], c.lens[2] = 1, 0
    c.run(ctx)
    torch.cuda.synchronize()
    assert bool((c.out[:3, :256] == 0).all()) and bool((c.out[12:14, :256] == 0).all())
    c.ids, c.ctxs, c.counts, c.cu = c.ids[1:2], c.ctxs[1:2], c.counts[1:2], c.cu[1:3]
    c.mask, keep = None if c.mask is None else c.mask, c.rows
    c.rows = c.cu[-1]
    k = c.out[c.rows:keep].clone()
    c.out[c.rows:keep] = 7
    c.check()
    assert bool((k[:, :256] == 0).all())


@pytest.mark.parametrize("dtype,q32,dim,n", [("f16", False, 64, 2), ("bf16", False, 128, 2), ("f16", False, 128, 70), ("f32", True, 64, 2), ("f32", True, 128, 9), ("f32", True, 40, 2)])
def test_an_infinite_value_of_next_to_no_weight(ctx, dtype, q32, dim, n):
    """The parts that hold the rows' own tokens have weights below 2^-149 when they are joined; an infinite value there still shows, as in the formula."""
    c = Case([3000], [n], 4, 1, dim, dtype, 16, mask="chain", q32=q32, seed=8)
    c.q[:, :4 * dim] = c.q[:, :4 * dim].abs() + 1
    for tok in range(2000, 3000 + n):
        c.k[c.layer, int(c.blocks[0, tok // 16]), tok % 16] = -20
    c.v[c.layer, int(c.blocks[0, 3000 // 16]), 3000 % 16, :, 5] = float("inf")
    c.run(ctx)
    c.check()


def test_32_bit_calls_on_two_streams_and_two_graphs_of_one_work_area(ctx):
    """Units are joined by whoever arrives last: objects of their own at the same time, and graphs that share one object one after the other."""
    cases = [Case([4000, 900], [7, 3], 8, 2, 128, "f32", 16, mask="tree", seed=1, q32=True), Case([2500, 1900], [5, 30], 8, 2, 64, "f16", 16, mask="tree", seed=2, q32=True)]
    s, ops, first = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None], []
    torch.cuda.synchronize()
    for rnd in range(6):
        for c in cases:
            c.out.fill_(7)
        torch.cuda.synchronize()
        for i, c in enumerate(cases):
            ops[i] = c.run(ctx, ops[i], s=s[i].cuda_stream)
        torch.cuda.synchronize()
        if rnd == 0:
            first = [c.out.clone() for c in cases]
            for c in cases:
                c.check()
        assert all(torch.equal(c.out, f) for c, f in zip(cases, first))
    # two calls of different shapes through one work area, each in a graph
    c, d = cases[0], Case([700, 60], [40, 1], 8, 2, 128, "f32", 16, mask="any", seed=5, q32=True)
    op = backend.TreeAttention(ctx, c.kv, 8)
    other = backend.TreeAttention(ctx, d.kv, 8)
    other._a.d_work = op._a.d_work
    graphs = []
    for x, o in ((c, op), (d, other)):
        x.run(ctx, o, s=s[0].cuda_stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s[0]):
            o.run_dev(x.layer, x.q.data_ptr(), x.out.data_ptr(), x.rows + x.pad, 2, x.d[0].data_ptr(), x.d[1].data_ptr(), x.d[2].data_ptr(), x.max_blocks,
                      d_mask=x.d[4].data_ptr(), mask_words=x.words, d_ids=x.d[3].data_ptr(), n_table=2, q_stride=x.qs, out_stride=x.os, stream=s[0].cuda_stream)
        graphs.append(g)
    for _ in range(4):
        c.out.fill_(7), d.out.fill_(7)
        torch.cuda.synchronize()
        with torch.cuda.stream(s[0]):
            graphs[0].replay()
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, first[0])
        d.check()


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,n", [("f16", 64, 4, 1, 2), ("bf16", 128, 8, 2, 70), ("f16", 128, 6, 2, 9)])
def test_a_wait_that_runs_out_ends_the_call_with_a_status(ctx, dtype, dim, heads, kv_heads, n):
    """With a limit of no time at all the warps that enqueue loads and products give up where they would wait, with some of them under way, and the others
    after their second: the call ends, the host learns of it, and the next call gives what the one before gave."""
    c = Case([4000, 900, 20], [n, 3, 1], heads, kv_heads, dim, dtype, 16, mask="tree", seed=1)
    op = c.run(ctx)
    c.check()
    first = c.out.clone()
    for _ in range(2):
        ctx.debug_set("tree_wait_cycles", 0)
        try:
            c.run(ctx, op)
            torch.cuda.synchronize()
            with pytest.raises(backend.UllmError) as e:
                ctx.synchronize()
            assert e.value.code == backend.ERR_TIMEOUT
        finally:
            ctx.debug_set("tree_wait_cycles", -1)
        c.out.fill_(7)
        c.run(ctx, op)
        torch.cuda.synchronize()
        ctx.synchronize()
        assert torch.equal(c.out, first)


STALE = """
import torch
import test_tree_attn_gpu as t
from ullm_b200 import backend
ctx = backend.CudaContext(0)
c = t.Case([2500, 300, 0], [7, 40, 1], 8, 2, 64, "f32", 16, mask="tree", q32=True, seed=3)
op = backend.TreeAttention(ctx, c.kv, c.heads, dtype=c.qd)
work = torch.empty(op._a.work_bytes // 8 + 1, dtype=torch.int64, device="cuda")
op._a.d_work = work.data_ptr()
first = None
for i in range(1, 9):
    for n in (1, 2):
        work.fill_((2 * i - 2 + n) << 16 | n)
        c.out.fill_(7)
        c.run(ctx, op)
        c.check()
        first = c.out.clone() if first is None else first
        assert torch.equal(c.out, first), (i, n)
print("equal")
"""


def test_numbers_left_in_a_work_area_are_no_counts(ctx):
    """64-bit numbers of the size of token ids and slots, over the first calls of a process: a count beside the number of a call looked like that once."""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(here), here, os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", STALE], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stdout + r.stderr[-2000:]


@pytest.mark.parametrize("dtype,dim,rows", [("f32", 64, 1), ("f32", 64, 5), ("f32", 128, 1), ("f32", 128, 9), ("f16", 64, 1), ("bf16", 128, 5), ("f32", 80, 2)])
def test_32_bit_sums_over_long_contexts_do_not_drift(ctx, dtype, dim, rows):
    """Sums of positive values over 32,000 tokens: each is off by no more than its roundings, and all of them together are not off to one side, as they are where
    every addition cuts off instead of rounding (with 100 blocks to a CTA that was 3 to 7e-6, always too small)."""
    n_seq, heads, kv_heads, ps, length = 8, 16, 8, 64, 32000
    per = -(-(length + rows) // ps)
    n_pages = n_seq * per
    g = torch.Generator(device="cuda").manual_seed(dim + rows)
    shape = (1, n_pages, ps, kv_heads, dim)
    k = torch.randn(shape, generator=g, device="cuda").mul(0.2).to(DT[dtype][1])
    v = torch.rand(shape, generator=g, device="cuda").add(0.5).to(DT[dtype][1])
    kv = backend.KvPages(DT[dtype][0], 1, n_pages, ps, kv_heads, dim, k.data_ptr(), v.data_ptr())
    total = n_seq * rows
    q = torch.randn((total, heads, dim), generator=g, device="cuda")
    out = torch.empty_like(q)
    blocks = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).view(n_seq, per)
    cu, lens = ints(np.arange(n_seq + 1) * rows), ints(np.full(n_seq, length + rows))
    op = backend.TreeAttention(ctx, kv, heads, dtype=backend.F32)
    op.run_dev(0, q.data_ptr(), out.data_ptr(), total, n_seq, cu.data_ptr(), lens.data_ptr(), blocks.data_ptr(), per, stream=stream())
    torch.cuda.synchronize()
    apart = []
    worst = 0.0
    for b in range(n_seq):
        kk, vv = (p[0, blocks[b].long()].reshape(per * ps, kv_heads, dim)[:length + rows].double() for p in (k, v))
        qq = q[b * rows:(b + 1) * rows].double().view(rows, kv_heads, heads // kv_heads, dim)
        s = torch.einsum("rhgd,khd->hgrk", qq, kk) * paged_ref.default_scale(dim)
        keys, me = torch.arange(length + rows, device="cuda"), torch.arange(rows, device="cuda")
        s = s.masked_fill(keys[None] > length + me[:, None], -float("inf"))
        ref = torch.einsum("hgrk,khd->rhgd", torch.softmax(s, -1), vv).reshape(rows, heads, dim)
        rel = (out[b * rows:(b + 1) * rows].double() - ref) / ref
        apart.append(rel.flatten())
        worst = max(worst, float(rel.abs().max()))
    # One value: a score (below 2.5 in magnitude, dim products) and its power of two, 2 (dim + 4) 2.5 + 8 half steps of 2^-23 for numerator and sum; the blocks of a
    # segment one after the other, its warps and the parts of a unit, at most 32000 / 32 + 8 + 296 additions, again twice.
    assert worst <= (5 * (dim + 4) + 8 + 2 * (32000 / 32 + 8 + 296)) * 2.0 ** -24
    # All values: additions that round to nearest are off to either side, and so are scores and weights, on which the values do not depend: over
    # `total * heads * dim` values (8,192 at least) nothing is left of them.  What is cut off always has one sign: within a block four sums of its size at most (two
    # tiles of keys, three products each, of which the first two come before there is a sum), a step of 2^-23 each; and where the two parts of a value end, on average half a unit of the lower part's
    # 11 bits, below 2^-21 of the value.
    assert abs(float(torch.cat(apart).mean())) <= 6 * 2.0 ** -23 + 2.0 ** -22


@pytest.mark.parametrize("dtype,q32,dim,n", [("f16", False, 64, 3), ("f16", False, 128, 70), ("bf16", False, 128, 3), ("bf16", False, 64, 150), ("f16", False, 40, 3), ("bf16", False, 96, 9),
                                             ("f32", True, 40, 3), ("f32", True, 64, 3), ("f32", True, 128, 40), ("f16", True, 64, 3)])
def test_infinite_values_of_committed_tokens_under_any_weight(ctx, dtype, q32, dim, n):
    """Committed tokens whose weights are 2^-50 and 2^-170 of the largest (zeros in 16 or 32 bits) hold infinities and a NaN: the row has them all the same.
    A key whose score is -inf has no weight at all, and 0 * inf is NaN."""
    c = Case([600, 4000, 3], [n, 2, 1], 4, 2, dim, dtype, 16, mask="any", seed=9, q32=q32)
    c.q[:, :4 * dim] = 1
    at = lambda b, tok: (c.layer, int(c.blocks[b, tok // 16]), tok % 16)
    for b, total in ((0, 600 + n), (1, 4002)):
        for tok in range(total):
            c.k[at(b, tok)] = 0
    low = lambda power: power / (1.4427 * dim ** 0.5)  # key whose score is 2^power of the others'
    for b, tok, power, col, value in ((0, 100, -50, 1, "inf"), (0, 200, -170, 2, "-inf"), (0, 301, -170, 3, "nan"), (0, 302, -50, 4, "inf"), (0, 450, -50, 4, "-inf"), (1, 17, -170, 5, "inf"),
                                      (1, 3999, -50, 6, "-inf"), (1, 2200, -170, 33, "inf")):
        c.k[at(b, tok)] = low(power)
        c.v[at(b, tok)][:, col] = float(value)
    for tok in range(0, 1500):  # the first blocks of a long context weigh next to nothing
        c.k[at(1, tok)] = low(-170)
    c.k[at(1, 2300)][1, 0] = -float("inf")
    c.v[at(1, 2300)][:, 7] = float("inf")
    c.run(ctx)
    c.check()


@pytest.mark.parametrize("dim,n", [(64, 2), (128, 3), (128, 70), (96, 2)])
def test_the_largest_bf16_values(ctx, dim, n):
    """A value at the end of the range under a weight of nearly one, in a block behind those whose scores are a few powers of two lower: the result is finite."""
    n_seq = 60
    c = Case([900] * n_seq, [n] * n_seq, 8, 4, dim, "bf16", 16, mask="tree", seed=dim)
    big = torch.finfo(torch.bfloat16).max
    c.q[:, :8 * dim] = 1
    for pool in (c.k, c.v):  # (what no sequence uses stays NaN)
        pool[c.layer] = pool[c.layer] * 0
    for b in range(n_seq):
        for tok, power, value in ((100, 0.0, -big), (600, 7.5, big)):  # the second one's score is 2^7.5 of the others'
            page, slot = int(c.blocks[b, tok // 16]), tok % 16
            c.k[c.layer, page, slot] = power / (1.4427 * dim ** 0.5)
            c.v[c.layer, page, slot, b % 4, 7 + (tok == 100)] = value
    c.run(ctx)
    c.check()


@pytest.mark.parametrize("dtype,q32", [("f16", False), ("bf16", False), ("f32", True)])
def test_many_chains_of_any_length(ctx, dtype, q32):
    """More than a window of 32 sequences without a mask, prompts of hundreds of rows in the later windows among single rows and empty entries."""
    rng = np.random.default_rng(12)
    counts = [int(x) for x in rng.integers(0, 3, 75)]
    ctxs = [int(x) for x in rng.integers(0, 200, 75)]
    for b, n in ((3, 150), (31, 40), (32, 290), (33, 0), (50, 131), (74, 270)):
        counts[b] = n
    for heads, kv_heads in ((4, 1), (4, 2)):
        c = Case(ctxs, counts, heads, kv_heads, 64, dtype, 16, mask="chain", seed=3, q32=q32)
        c.run(ctx)
        c.check()


@pytest.mark.parametrize("dtype,q32,dim", [("f16", False, 64), ("bf16", False, 128), ("f32", True, 64), ("f16", True, 128), ("f32", True, 40)])
def test_a_row_of_infinitely_low_scores_becomes_zeros(ctx, dtype, q32, dim):
    """As a row that sees nothing; the other sequences are what they were."""
    c = Case([300, 50], [5, 3], 4, 2, dim, dtype, 16, mask="tree", seed=4, q32=q32)
    c.q[:, :4 * dim] = c.q[:, :4 * dim].abs() + 0.1
    c.run(ctx)
    torch.cuda.synchronize()
    before = c.out.clone()
    for tok in range(305):
        c.k[c.layer, int(c.blocks[0, tok // 16]), tok % 16, :, 1] = -float("inf")
    c.run(ctx)
    torch.cuda.synchronize()
    assert bool((c.out[:5, :4 * dim] == 0).all()) and torch.equal(c.out[5:], before[5:])
