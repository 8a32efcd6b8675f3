"""GPU tests of the tables of a paged cache, the plan of a step and the norm + rotation + cache write, against the rules of
paged_ref.py in 64 bits."""
import numpy as np
import pytest
import torch

import paged_ref
from ullm_b200 import backend

pytestmark = pytest.mark.gpu
DT = {"f32": (backend.F32, torch.float32), "f16": (backend.F16, torch.float16), "bf16": (backend.BF16, torch.bfloat16)}


def ints(v):
    return torch.as_tensor(np.asarray(v, np.int32)).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def make_pool(layers, n_pages, ps, heads, dim, dtype, layout, seed, spare=0):
    """K, V seen as [layer, page, slot, head, dim] and their description; `spare`: values between two heads."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        shape = (layers, n_pages, ps, heads, dim + spare) if layout == "slot" else (layers, n_pages, heads, ps, dim + spare)
        t = torch.randn(shape, generator=g).to(DT[dtype][1]).cuda()[..., :dim]
        out.append(t if layout == "slot" else t.transpose(2, 3))
    k, v = out
    st = k.stride()
    kv = backend.KvPages(DT[dtype][0], layers, n_pages, ps, heads, dim, k.data_ptr(), v.data_ptr(), strides=st[:4])
    return k, v, kv


class Both:
    """The library's tables beside the reference's."""

    def __init__(self, ctx, n_seq, max_blocks, n_pages, ps, layers=2, heads=2, dim=16, dtype="f16", layout="slot", seed=1, spare=0):
        self.k, self.v, self.kv = make_pool(layers, n_pages, ps, heads, dim, dtype, layout, seed, spare)
        self.ref = paged_ref.Tables(n_seq, max_blocks, n_pages, ps, self.k.cpu().float().numpy(), self.v.cpu().float().numpy())
        self.blocks, self.len = ints(np.full((n_seq, max_blocks), -7)), ints(np.zeros(n_seq))
        self.refs, self.fault = ints(np.zeros(n_pages)), ints([0])
        self.t = backend.KvTable(ctx, self.kv, self.blocks.data_ptr(), self.len.data_ptr(), self.refs.data_ptr(), self.fault.data_ptr(), n_seq, max_blocks)

    def call(self, name, *lists):
        arrays = [None if a is None else ints(a) for a in lists]
        ptrs = [None if a is None else a.data_ptr() for a in arrays]
        n = len(lists[0])
        getattr(self.t, name + "_dev")(*ptrs, n, *([arrays[2].shape[1]] if name == "accept" else []), stream=stream())
        torch.cuda.synchronize()
        getattr(self.ref, name)(*[None if a is None else np.asarray(a) for a in lists])
        self.check()

    def put(self, blocks=None, length=None, refs=None):
        for dev, ref, new in ((self.blocks, self.ref.blocks, blocks), (self.len, self.ref.len, length), (self.refs, self.ref.refs, refs)):
            if new is not None:
                ref[...] = new
                dev.copy_(ints(new))

    def check(self):
        r = self.ref
        assert int(self.fault[0]) == r.fault
        assert np.array_equal(self.len.cpu().numpy(), r.len)
        assert np.array_equal(self.refs.cpu().numpy(), r.refs)
        assert np.array_equal(self.blocks.cpu().numpy(), r.blocks)
        for got, ref in ((self.k, r.k), (self.v, r.v)):
            differ = int((got.cpu().float().numpy() != ref).sum())
            assert differ == 0

    def clear(self):
        self.fault.zero_()
        self.ref.fault = 0


@pytest.mark.parametrize("n_seq,n_pages,ps,dtype,layout,dim,spare,seed", [
    (1, 3, 4, "f16", "slot", 16, 0, 0), (5, 40, 1, "f32", "slot", 8, 0, 1), (6, 60, 3, "bf16", "head", 24, 8, 2), (16, 300, 16, "f16", "head", 64, 0, 3),
    (40, 3000, 2, "bf16", "slot", 8, 0, 4), (7, 9000, 5, "f16", "slot", 8, 0, 5),
])
def test_random_life_of_a_pool(ctx, n_seq, n_pages, ps, dtype, layout, dim, spare, seed):
    """Every operation in random order; refused entries included.  All values are copies, so everything is equal."""
    rng = np.random.default_rng(seed)
    b = Both(ctx, n_seq, 12, n_pages, ps, dtype=dtype, layout=layout, dim=dim, spare=spare, seed=seed)
    for step in range(30):
        op = rng.choice(["grow", "grow", "fork", "accept", "trim"])
        m = int(rng.integers(1, n_seq + 1))
        rows = rng.permutation(n_seq)[:m]
        if rng.random() < 0.15:
            rows[rng.integers(m)] = rng.choice([-1, n_seq, rows[0]])
        if op == "grow":
            b.call("grow", rows, rng.integers(-1 if rng.random() < 0.1 else 0, 3 * ps + 2, m))
        elif op == "fork":
            b.call("fork", rng.integers(0, n_seq, m), rows)
        elif op == "trim":
            new = [int(rng.integers(0, b.ref.len[r] + (2 if rng.random() < 0.1 else 1))) if 0 <= r < n_seq else 0 for r in rows]
            b.call("trim", rows, None if rng.random() < 0.3 else new)
        else:
            draft = np.array([int(rng.integers(0, min(b.ref.len[r], 20) + 1)) if 0 <= r < n_seq else 1 for r in rows])
            path, kept = np.zeros((m, 24), int), np.array([int(rng.integers(0, d + 1)) for d in draft])
            for i in range(m):
                path[i, :kept[i]] = np.sort(rng.choice(draft[i], kept[i], replace=False))
                if rng.random() < 0.1 and kept[i] > 1:
                    path[i, :2] = path[i, 1]
            b.call("accept", rows, draft, path, kept)
        if rng.random() < 0.5:
            b.clear()


def test_pages_run_out_without_a_trace(ctx):
    b = Both(ctx, 4, 8, 10, 4)
    b.call("grow", [0, 1], [9, 20])
    assert b.ref.fault == 0
    b.call("grow", [2, 3, 0], [4, 4, 1])  # the last two pages; row 0 still has room in its third
    assert b.ref.fault == 0
    b.call("grow", [2, 3], [1, 1])
    assert b.ref.fault == backend.KV_FAULT_NO_PAGES


def test_corrupt_tables_are_reported_not_followed(ctx):
    b = Both(ctx, 4, 8, 10, 4)
    b.call("grow", [0, 1, 2], [10, 10, 6])
    bad = b.ref.blocks.copy()
    bad[0, 2], bad[1, 0], bad[2, 1] = 10, -1, 1 << 30
    b.put(blocks=bad)
    b.call("fork", [0, 1], [3, 3])
    b.call("fork", [1], [3])
    assert b.ref.fault & backend.KV_FAULT_PAGE
    b.clear()
    b.call("grow", [2], [1])
    assert b.ref.fault == backend.KV_FAULT_PAGE
    b.clear()
    b.call("accept", [0], [6], [[3, 5]], [2])
    assert b.ref.fault == backend.KV_FAULT_PAGE
    b.clear()
    b.call("trim", [0, 1, 2], None)
    assert b.ref.fault == backend.KV_FAULT_PAGE
    b.clear()
    b.put(length=[-3, 1000, 33, 0])
    b.call("fork", [0, 1], [3, 3])
    b.call("fork", [1], [3])
    b.call("grow", [0, 1, 2], [1, 1, 1])
    b.call("trim", [0, 1, 2], [0, 0, 0])
    b.call("accept", [0, 1, 2], [1, 1, 1], [[0], [0], [0]], [1, 1, 1])
    assert b.ref.fault == backend.KV_FAULT_LEN | backend.KV_FAULT_SEQ


def test_copy_pages(ctx):
    for layout in ("slot", "head"):
        b = Both(ctx, 1, 1, 12, 5, layers=3, dim=40, layout=layout, spare=8)
        src, dst = [3, 4, 11, 12, 0, 5, 6, 1], [0, 7, 8, 9, 2, 10, 10, -1]
        d_src, d_dst = ints(src), ints(dst)
        b.t.copy_pages_dev(d_src.data_ptr(), d_dst.data_ptr(), len(src), stream=stream())
        torch.cuda.synchronize()
        for s, d in ((4, 7), (11, 8), (0, 2)):  # 3 -> 0 would change a source, 12 and -1 are no pages, 10 is asked for twice
            b.ref.k[:, d], b.ref.v[:, d] = b.ref.k[:, s], b.ref.v[:, s]
        b.ref.fault = backend.KV_FAULT_PAGE
        b.check()


def test_a_captured_step_replays_on_what_the_tables_then_hold(ctx):
    b = Both(ctx, 4, 16, 64, 4, layers=3)
    b.call("grow", [0], [6])
    seq, add, src, dst = ints([0, 1]), ints([5, 5]), ints([0]), ints([1])
    path, kept = ints([[1, 3, 0], [0, 2, 4]]), ints([2, 3])
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st = s.cuda_stream
        b.t.fork_dev(src.data_ptr(), dst.data_ptr(), 1, stream=st)
        b.t.grow_dev(seq.data_ptr(), add.data_ptr(), 2, stream=st)
        b.t.accept_dev(seq.data_ptr(), add.data_ptr(), path.data_ptr(), kept.data_ptr(), 2, 3, stream=st)
        b.t.trim_dev(dst.data_ptr(), None, 1, stream=st)
    b.check()  # nothing has run
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        b.ref.fork([0], [1])
        b.ref.grow([0, 1], [5, 5])
        b.ref.accept([0, 1], [5, 5], np.array([[1, 3, 0], [0, 2, 4]]), [2, 3])
        b.ref.trim([1])
        b.check()
    assert b.ref.fault == 0 and b.ref.len[0] == 14


@pytest.mark.parametrize("lens,counts,words,pad,chain,ids", [
    ([1], [1], 1, 0, False, None), ([40, 7, 200], [33, 0, 64], 2, 5, False, None), ([40, 7, 200], [33, 7, 64], 0, 1, False, None),
    ([300, 9, 4], [100, 9, 4], 4, 2, True, None), ([5, 130, 60], [129, 20], 5, 700, False, [1, 2]), ([10, 10, 500], [12, 10, 400], 4, 3, False, None),
    ([9, 9], [3, 4], 1, 0, False, [1, 7]),
])
def test_plan(ctx, lens, counts, words, pad, chain, ids):
    rng = np.random.default_rng(len(lens) + sum(counts))
    cu = np.concatenate([[0], np.cumsum(counts)])
    rows = int(cu[-1]) + pad
    parents = None if chain else np.concatenate([paged_ref.tree_parents(n, rng) for n in counts] + [np.full(pad, 99)])
    if parents is not None and counts[0] > 4:
        parents[3], parents[4] = 3, -2  # no node in front of them: they hang on the last committed token
    want = paged_ref.plan(cu, lens, parents, rows, words or None, ids)
    d_cu, d_len, d_par = ints(cu), ints(lens), None if chain else ints(parents)
    seq, slot, pos = (ints(np.full(rows, -9)) for _ in range(3))
    mask = torch.full((rows, max(words, 1)), -286331154, dtype=torch.int32, device="cuda")  # 0xEEEEEEEE
    fault, d_ids = ints([0]), None if ids is None else ints(ids)
    ctx.tree_plan_dev(rows, len(counts), d_cu.data_ptr(), d_len.data_ptr(), None if chain else d_par.data_ptr(), seq.data_ptr(), slot.data_ptr(), pos.data_ptr(),
                      mask.data_ptr() if words else None, words, fault.data_ptr(), None if ids is None else d_ids.data_ptr(), len(lens), stream())
    torch.cuda.synchronize()
    for got, ref in zip((seq, slot, pos), want):
        assert np.array_equal(got.cpu().numpy(), ref)
    assert np.array_equal(mask.cpu().numpy().view(np.uint32), want[3])
    assert int(fault[0]) == want[4]


@pytest.mark.parametrize("x,dtype,q32,heads,kv_heads,dim,rot,ps,layout,norm,bias,neox,rows", [
    ("f32", "f16", False, 4, 2, 64, 0, 16, "slot", False, False, False, 1),
    ("f32", "f16", True, 8, 8, 128, 0, 32, "head", True, False, True, 13),
    ("bf16", "bf16", False, 5, 1, 128, 64, 7, "slot", True, True, True, 300),
    ("f16", "f16", False, 6, 3, 16, 0, 1, "slot", True, True, False, 37),
    ("f32", "f32", True, 4, 4, 256, 0, 4, "head", True, False, True, 21),
    ("bf16", "f32", True, 3, 1, 96, 96, 16, "slot", True, True, True, 50),
    ("f16", "bf16", False, 2, 2, 40, 32, 5, "head", False, True, True, 19),
    ("f32", "bf16", False, 32, 4, 128, 0, 64, "slot", True, False, True, 130),
    ("f32", "bf16", True, 7, 7, 24, 16, 3, "slot", True, False, False, 5),
])
def test_norm_rotation_and_cache_write(ctx, x, dtype, q32, heads, kv_heads, dim, rot, ps, layout, norm, bias, neox, rows):
    rng = np.random.default_rng(rows)
    rot_n, pad, n_seq, layers = rot or dim, 3, 3, 2
    max_blocks = -(-rows // ps) + 2
    k, v, kv = make_pool(layers, n_seq * max_blocks + 2, ps, kv_heads, dim, dtype, layout, rows, spare=8 if dim % 16 else 0)
    blocks = rng.permutation(n_seq * max_blocks + 2)[:n_seq * max_blocks].reshape(n_seq, max_blocks)
    total = rows + pad
    seq = np.concatenate([rng.integers(0, n_seq, rows), np.full(pad, -1)])
    slot = np.concatenate([rng.permutation(max_blocks * ps)[:rows], np.full(pad, 10 ** 6)])  # rows meet in no slot
    n_pos = 50
    pos = np.concatenate([rng.integers(0, n_pos, rows), np.full(pad, -5)])
    width = (heads + 2 * kv_heads) * dim + 16
    xs = torch.randn(total, width, generator=torch.Generator().manual_seed(rows)).mul(1.5).to(DT[x][1]).cuda()
    angle = np.arange(n_pos)[:, None] * 1e4 ** (-np.arange(rot_n // 2) / (rot_n // 2))[None]
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    w = [1 + 0.1 * rng.standard_normal(dim).astype(np.float32) for _ in range(2)] if norm else [None, None]
    bs = [rng.standard_normal(n * dim).astype(np.float32) for n in (heads, kv_heads, kv_heads)] if bias else [None] * 3
    dev = [None if a is None else torch.as_tensor(a).cuda() for a in (*w, *bs, cs)]
    ptr = [None if a is None else a.data_ptr() for a in dev]
    qt = torch.float32 if q32 else DT[dtype][1]
    q = torch.full((total, heads * dim + 32), 7.0, dtype=qt, device="cuda")
    k0, v0 = k.clone(), v.clone()
    op = backend.QkNormRope(ctx, kv, heads, DT[x][0], ptr[5], n_pos, q_dtype=backend.F32 if q32 else DT[dtype][0], rot_dim=rot, neox=neox, d_q_norm=ptr[0],
                            d_k_norm=ptr[1], eps=1e-5, d_q_bias=ptr[2], d_k_bias=ptr[3], d_v_bias=ptr[4])
    e = xs.element_size()
    fault = ints([0])
    lists = [ints(a) for a in (pos, seq, slot, blocks)]
    op.run_dev(1, xs.data_ptr(), xs.data_ptr() + heads * dim * e, xs.data_ptr() + (heads + kv_heads) * dim * e, q.data_ptr(), total, *[a.data_ptr() for a in lists],
               n_seq, max_blocks, x_stride=width, q_out_stride=heads * dim + 32, d_fault=fault.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert int(fault[0]) == 0
    h = xs[:rows].double().cpu().numpy()
    parts = [h[:, :heads * dim], h[:, heads * dim:(heads + kv_heads) * dim], h[:, (heads + kv_heads) * dim:(heads + 2 * kv_heads) * dim]]
    parts = [a if b is None else a + b for a, b in zip(parts, bs)]
    c = cs.astype(np.float64)[pos[:rows]]
    page, at = blocks[seq[:rows], slot[:rows] // ps], slot[:rows] % ps
    # f32: bias 1, sum of squares dim / 8 + 5, mean, eps, root, quotient, two products, two products and a sum of the rotation: under 16 + dim / 16 half steps of
    # 2^-24 each on the magnitudes that are added; then one rounding to the type, half a step of the value
    tol32 = (16 + dim / 16) * 2.0 ** -24
    for name, got, src, n_heads, weight in (("q", q[:rows, :heads * dim], parts[0], heads, w[0]), ("k", k[1], parts[1], kv_heads, w[1]), ("v", v[1], parts[2], kv_heads, None)):
        if name == "v":
            ref = src.reshape(rows, n_heads, dim)
            mag = np.abs(ref)
        else:
            ref, mag = paged_ref.rope_rows(src, n_heads, weight, 1e-5, c, rot_n, neox)
        got = got if name == "q" else got[torch.as_tensor(page).cuda(), torch.as_tensor(at).cuda()]
        half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
        err = np.abs(got.double().cpu().numpy().reshape(ref.shape) - ref)
        bound = half * np.abs(ref) * (1 + tol32) + tol32 * mag + np.abs(src).max() * 1e-30 + (6e-8 if got.dtype == torch.float16 else 0.0)  # f16: half a subnormal step
        assert (err <= bound).all(), (name, float((err / np.maximum(bound, 1e-300)).max()))
    # what is not the rows' stays as it was
    assert bool((q[rows:] == 7).all()) and bool((q[:, heads * dim:] == 7).all())
    for new, old in ((k, k0), (v, v0)):
        old[1, torch.as_tensor(page).cuda(), torch.as_tensor(at).cuda()] = new[1, torch.as_tensor(page).cuda(), torch.as_tensor(at).cuda()]
        assert torch.equal(new, old)


def test_rope_in_place_and_rows_outside_are_left_out(ctx):
    heads, kv_heads, dim, ps, rows = 4, 2, 64, 8, 6
    k, v, kv = make_pool(1, 4, ps, kv_heads, dim, "f16", "slot", 3)
    k0, v0 = k.clone(), v.clone()
    x = torch.randn(rows, (heads + 2 * kv_heads) * dim, generator=torch.Generator().manual_seed(4)).half().cuda()
    x0 = x.clone()
    cs = torch.randn(10, dim // 2, 2, generator=torch.Generator().manual_seed(5)).cuda()
    blocks = ints([[0, 9], [2, -1]])
    seq, slot, pos = ints([0, 0, 1, 1, 2, 0]), ints([0, 8, 3, 8, 0, 16]), ints([3, 3, 10, 3, 3, 3])
    fault = ints([0])
    op = backend.QkNormRope(ctx, kv, heads, backend.F16, cs.data_ptr(), 10)
    p = x.data_ptr()
    op.run_dev(0, p, p + heads * dim * 2, p + (heads + kv_heads) * dim * 2, p, rows, pos.data_ptr(), seq.data_ptr(), slot.data_ptr(), blocks.data_ptr(), 2, 2,
               x_stride=x.shape[1], q_out_stride=x.shape[1], d_fault=fault.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert int(fault[0]) == backend.KV_FAULT_PAGE | backend.KV_FAULT_POS | backend.KV_FAULT_LEN
    assert torch.equal(x[1:], x0[1:]) and not torch.equal(x[0, :heads * dim], x0[0, :heads * dim]) and torch.equal(x[0, heads * dim:], x0[0, heads * dim:])
    ref, mag = paged_ref.rope_rows(x0[:1, :heads * dim].double().cpu().numpy(), heads, None, 0, cs[3:4].double().cpu().numpy(), dim, False)
    err = np.abs(x[:1, :heads * dim].double().cpu().numpy().reshape(ref.shape) - ref)
    assert (err <= 2.0 ** -11 * np.abs(ref) + 4 * 2.0 ** -24 * mag + 6e-8).all()
    k0[0, 0, 0], v0[0, 0, 0] = k[0, 0, 0], v[0, 0, 0]
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_lengths_at_the_ends_of_the_range_are_refused(ctx):
    """Counting such a length in pages would pass 32 bits; every call refuses it before it looks into the table."""
    for ps in (16, 5):
        b = Both(ctx, 6, 8, 10, ps)
        b.call("grow", [0], [ps + 3])
        top, low = 2 ** 31 - 1, -(2 ** 31)
        b.put(length=[ps + 3, top, top - 1, low, low + 1, 0])
        for s in (1, 2, 3, 4):
            for name, lists in (("fork", ([s], [5])), ("trim", ([s], [0])), ("trim", ([s], None)), ("accept", ([s], [4], [[1, 3]], [2])), ("accept", ([s], [top], [[top - 1]], [1])),
                                ("grow", ([s], [1]))):
                b.call(name, *lists)
                assert b.ref.fault == backend.KV_FAULT_LEN
                b.clear()
        b.call("accept", [0], [3], [[0, 2]], [2])
        assert b.ref.fault == 0


def test_plan_refuses_lengths_at_the_ends_of_the_range(ctx):
    lens = [2 ** 31 - 1, -(2 ** 31), -(2 ** 31) + 3, 9]
    cu, rows = [0, 3, 7, 9, 11], 12
    want = paged_ref.plan(cu, lens, None, rows, 1)
    d = [ints(a) for a in (cu, lens)]
    seq, slot, pos = (ints(np.full(rows, -9)) for _ in range(3))
    mask, fault = torch.full((rows, 1), -286331154, dtype=torch.int32, device="cuda"), ints([0])
    ctx.tree_plan_dev(rows, 4, d[0].data_ptr(), d[1].data_ptr(), None, seq.data_ptr(), slot.data_ptr(), pos.data_ptr(), mask.data_ptr(), 1, fault.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert seq.tolist() == [0] * 3 + [-1] * 6 + [3] * 2 + [-1] and int(fault[0]) == want[4] == backend.KV_FAULT_LEN
    assert np.array_equal(slot.cpu().numpy(), want[1]) and np.array_equal(pos.cpu().numpy(), want[2]) and np.array_equal(mask.cpu().numpy().view(np.uint32), want[3])


def test_wants_beyond_32_bits_are_refused_as_a_whole(ctx):
    """512 rows that ask for 2^22 pages each: the sum is 2^31 pages."""
    n, blocks, pages = 512, 1 << 22, 64
    k, v, kv = make_pool(1, pages, 1, 1, 8, "f16", "slot", 1)
    table = torch.empty((n, blocks), dtype=torch.int32, device="cuda")
    lens, refs, fault = ints(np.zeros(n)), ints(np.zeros(pages)), ints([0])
    t = backend.KvTable(ctx, kv, table.data_ptr(), lens.data_ptr(), refs.data_ptr(), fault.data_ptr(), n, blocks)
    seq = ints(np.arange(n))
    for add in (blocks, blocks - 1, 1 << 20):
        adds = ints(np.full(n, add))
        fault.zero_()
        t.grow_dev(seq.data_ptr(), adds.data_ptr(), n, stream=stream())
        torch.cuda.synchronize()
        assert int(fault[0]) == backend.KV_FAULT_NO_PAGES and int(lens.abs().sum()) == 0 and int(refs.sum()) == 0
    adds = ints(np.arange(n) < 60)
    fault.zero_()
    t.grow_dev(seq.data_ptr(), adds.data_ptr(), n, stream=stream())
    torch.cuda.synchronize()
    assert int(fault[0]) == 0 and int(lens.sum()) == 60 and torch.equal(table[:60, 0], torch.arange(60, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("cu,good", [([0, 5, 3, 8], False), ([0, 3, -1], False), ([-2, 3, 6], False), ([0, 4, 13], False), ([9, 4, 2], False), ([0, 2 ** 31 - 1, 5], False),
                                     ([-(2 ** 31), 2, 5], False), ([3, 5, 5, 9], True), ([12, 12], True), ([0, 0], True)])
def test_plan_leaves_no_row_stale(ctx, cu, good):
    """Rows that no sequence owns get -1, whatever the array held: a later cache write skips them.  Offsets out of order refuse all rows."""
    rows, n = 12, len(cu) - 1
    d_cu, d_len = ints(cu), ints([40] * n)
    seq, slot, pos = (ints(np.full(rows, 1)) for _ in range(3))
    fault = ints([0])
    ctx.tree_plan_dev(rows, n, d_cu.data_ptr(), d_len.data_ptr(), None, seq.data_ptr(), slot.data_ptr(), pos.data_ptr(), None, 0, fault.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    want = np.full(rows, -1)
    if good:
        for b in range(n):
            want[cu[b]:cu[b + 1]] = b
    assert seq.tolist() == want.tolist() and int(fault[0]) == (0 if good else backend.KV_FAULT_LEN)
    assert slot[np.nonzero(want < 0)[0].tolist()].eq(1).all() and pos[np.nonzero(want < 0)[0].tolist()].eq(1).all()


@pytest.mark.parametrize("cu,ids,want", [
    ([0, 3, 5], [2, 2], [-1] * 5), ([0, 3, 5, 8], [1, 0, 1], [-1] * 3 + [0] * 2 + [-1] * 3), ([0, 3, 5, 5, 5], [1, 0, 0, 1], [1] * 3 + [0] * 2), ([0, 0, 4, 4], [1, 1, 1], [1] * 4),
    ([0] + [200] * 300, [2] * 300, [2] * 200),
])
def test_plan_refuses_a_table_row_that_is_named_twice(ctx, cu, ids, want):
    """Two sequences cannot both be a row's last tokens.  Entries without rows (a padded batch) may name any row."""
    rows, n = cu[-1], len(ids)
    d_cu, d_len, d_ids = ints(cu), ints([400] * 3), ints(ids)
    seq, slot, pos = (ints(np.full(rows, -9)) for _ in range(3))
    fault = ints([0])
    ctx.tree_plan_dev(rows, n, d_cu.data_ptr(), d_len.data_ptr(), None, seq.data_ptr(), slot.data_ptr(), pos.data_ptr(), None, 0, fault.data_ptr(), d_ids.data_ptr(), 3, stream())
    torch.cuda.synchronize()
    assert seq.tolist() == want and int(fault[0]) == (backend.KV_FAULT_SEQ if -1 in want else 0)
