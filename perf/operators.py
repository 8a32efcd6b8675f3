"""Cases and plain forms of the operators over a paged key/value cache.

Four operators of one serving step, in the order in which the step uses them:

``pages``   the tables of a paged cache: sequences fork (share pages), grow (lowest free pages first, a shared page
            that is about to be written is copied first), keep the accepted rows of a drafted tree (rows move up,
            pages behind them are freed) and are released.
``plan``    a tree of drafted tokens, given as parents, turned into what the layers need: each row's sequence, slot
            and position, and the bits of the ancestors that it may see.
``rope``    RMS norms of each query and key head, the position rotation, and the rows' keys and values written into
            their pages, in one pass.
``attn``    attention of the drafted rows over their sequences' pages: all committed tokens, and among the drafted
            ones those that the row's bits name.  One token per sequence is ordinary decoding.

``run`` computes the plain forms with elementary torch operations in 32 bits; where ``own`` is true it makes the
library's calls instead.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    # (query heads, key heads, head dimension): 32/8/64 is the dense decode configuration, 32/4/128 the
    # mixture-of-experts one, 64/8/128 the large dense block.
    return [
        # one user, one token, about a thousand tokens of context: the latency of plain decoding
        dict(name="attn one token", op="attn", batch=1, draft=1, ctx_min=1100, ctx_max=1100, n_head=32, n_kv=8, dim=64, dtype="f16", page=16,
             layout="slot", pad=0, shape=1),
        # a small tree for each of eight users
        dict(name="attn small trees", op="attn", batch=8, draft=12, ctx_min=300, ctx_max=5000, n_head=32, n_kv=4, dim=128, dtype="bf16", page=32,
             layout="slot", pad=3, shape=2),
        # a full serving batch that decodes one token per user, contexts of very different length
        dict(name="attn batch decode", op="attn", batch=64, draft=1, ctx_min=100, ctx_max=8000, n_head=64, n_kv=8, dim=128, dtype="bf16", page=64,
             layout="head", pad=0, shape=3),
        # wide trees over long contexts: the largest arithmetic
        dict(name="attn wide trees", op="attn", batch=12, draft=64, ctx_min=4000, ctx_max=16000, n_head=64, n_kv=8, dim=128, dtype="f16", page=64,
             layout="slot", pad=5, shape=4),
        # one user, a very long context, a short draft
        dict(name="attn long context", op="attn", batch=1, draft=13, ctx_min=130001, ctx_max=130001, n_head=64, n_kv=8, dim=128, dtype="bf16", page=128,
             layout="slot", pad=0, shape=5),
        # the engine's default cache: all 32 bits
        dict(name="attn f32 cache", op="attn", batch=3, draft=7, ctx_min=500, ctx_max=2000, n_head=32, n_kv=8, dim=64, dtype="f32", page=16,
             layout="slot", pad=0, shape=6),
        # one decoded token of one user of the dense configuration: projections in 32 bits, cache in half precision
        dict(name="rope one token", op="rope", rows=1, batch=1, n_head=32, n_kv=8, dim=64, x="f32", dtype="f16", page=16, norm=False, neox=False,
             layout="slot", pad=0, shape=7),
        # a long prompt
        dict(name="rope prompt", op="rope", rows=16000, batch=4, n_head=64, n_kv=8, dim=128, x="bf16", dtype="bf16", page=64, norm=True, neox=True,
             layout="head", pad=3, shape=9),
        # a few users' speculative step: the tables' latency
        dict(name="pages few", op="pages", seqs=4, forks=4, draft=6, ctx_max=700, layers=4, n_kv=8, dim=64, dtype="f16", page=16, layout="slot", shape=10),
        # a serving batch in which every sequence branches
        dict(name="pages many", op="pages", seqs=96, forks=96, draft=24, ctx_max=900, layers=12, n_kv=4, dim=128, dtype="bf16", page=32, layout="slot",
             shape=11),
        # one user's tree
        dict(name="plan one tree", op="plan", batch=1, draft=8, ctx_max=1000, pad=0, shape=12),
        # the trees of a large batch
        dict(name="plan many trees", op="plan", batch=200, draft=61, ctx_max=9000, pad=11, shape=13),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["attn", "attn", "attn", "rope", "pages", "plan"])
    shape = rng.randrange(1 << 30)
    heads = rng.choice([(32, 8, 64), (32, 4, 128), (64, 8, 128), (8, 8, 64), (16, 1, 128), (9, 3, 64), (4, 4, 128)])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.choice(["slot", "head"])
    if op == "attn":
        h, k, d = heads
        batch, draft, ctx = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 16, 130000)
        # no more cached bytes and no more arithmetic than the largest listed cases
        most = 1.0e9 / (batch * 2 * k * d * BYTES[dtype])
        most = min(most, 3.0e11 * (0.02 if dtype == "f32" else 1.0) / (4.0 * batch * draft * h * d), 1.6e8 / (batch * draft * h))
        ctx = max(16, min(ctx, int(most)))
        lo = rng.choice([0, ctx // 10, ctx])
        return dict(op=op, batch=batch, draft=draft, ctx_min=lo, ctx_max=ctx, n_head=h, n_kv=k, dim=d, dtype=dtype, page=page, layout=layout,
                    pad=rng.choice([0, 0, 1, 7]), shape=shape)
    if op == "rope":
        h, k, d = heads
        rows = min(_log(rng, 1, 16000), int(16000 * 80 * 128 / ((h + 2 * k) * d)))
        return dict(op=op, rows=rows, batch=min(rows, _log(rng, 1, 64)), n_head=h, n_kv=k, dim=d, x=rng.choice(["f32", dtype]), dtype=dtype, page=page,
                    norm=rng.random() < 0.7, neox=rng.random() < 0.5, layout=layout, pad=rng.choice([0, 0, 1, 7]), shape=shape)
    if op == "pages":
        _, k, d = heads
        seqs, layers = _log(rng, 1, 96), rng.choice([1, 4, 12])
        ctx = _log(rng, 8, 900)
        return dict(op=op, seqs=seqs, forks=rng.randint(0, seqs), draft=_log(rng, 1, 32), ctx_max=ctx, layers=layers, n_kv=min(k, 4), dim=d,
                    dtype=rng.choice(["f16", "bf16"]), page=rng.choice([16, 32]), layout=layout, shape=shape)
    return dict(op=op, batch=_log(rng, 1, 200), draft=_log(rng, 1, 120), ctx_max=_log(rng, 1, 9000), pad=rng.choice([0, 1, 11]), shape=shape)


# ---------------------------------------------------------------------------------------------------------------
# What a case's lengths are (the same for every seed)
# ---------------------------------------------------------------------------------------------------------------
def _ragged(case):
    """Committed tokens and drafted rows of every sequence of an attention or plan case."""
    r = random.Random(case["shape"])
    lo, hi = case.get("ctx_min", 0), case["ctx_max"]
    ctx = [hi if lo == hi else int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))) - 1)) for _ in range(case["batch"])]
    n = [r.randint(max(1, (case["draft"] + 1) // 2), case["draft"]) for _ in range(case["batch"])]
    ctx[0], n[0] = hi, case["draft"]
    return ctx, n


def _rope_rows(case):
    """Rows of every sequence of a rope case (they sum to case['rows']) and the tokens in front of them."""
    r = random.Random(case["shape"])
    cut = sorted(r.sample(range(1, case["rows"]), case["batch"] - 1)) if case["batch"] > 1 else []
    n = [b - a for a, b in zip([0] + cut, cut + [case["rows"]])]
    return [r.randint(0, 200) for _ in n], n


def _page_lengths(case):
    r = random.Random(case["shape"])
    length = [r.randint(0 if case["seqs"] > 1 else 1, case["ctx_max"]) for _ in range(case["seqs"])]
    parent = [r.randrange(case["seqs"]) for _ in range(case["forks"])]
    add = [r.randint(1, case["draft"]) for _ in range(case["seqs"] + case["forks"])]
    return length, parent, add


def work(case):
    if case["op"] == "attn":
        ctx, n = _ragged(case)
        b, row = BYTES[case["dtype"]], case["n_head"] * case["dim"]
        keys = sum(c + k for c, k in zip(ctx, n))
        pairs = sum(k * (c + 1) for c, k in zip(ctx, n))
        words = (case["draft"] + 31) // 32
        return {"bytes": keys * case["n_kv"] * case["dim"] * 2 * b + sum(n) * (2 * row * b + 4 * words) + 4 * sum(-(-(c + k) // case["page"]) for c, k in zip(ctx, n)),
                "flops": 4.0 * case["dim"] * case["n_head"] * pairs}
    if case["op"] == "rope":
        q, kv = case["n_head"] * case["dim"], case["n_kv"] * case["dim"]
        per_row = (q + 2 * kv) * (BYTES[case["x"]] + BYTES[case["dtype"]]) + 12 + case["dim"] * 4
        return {"bytes": case["rows"] * per_row, "flops": case["rows"] * (q + kv) * (7.0 if case["norm"] else 3.0)}
    if case["op"] == "pages":
        length, parent, add = _page_lengths(case)
        row = 2 * case["layers"] * case["n_kv"] * case["dim"] * BYTES[case["dtype"]]
        shared = {p for p in parent}
        copied = sum(length[p] % case["page"] for p in shared) + sum(length[p] % case["page"] for p in parent)
        moved = sum(a // 2 for a in add)
        tables = 4 * sum(-(-(length[p] + case["draft"]) // case["page"]) for p in parent) * 3
        return {"bytes": 2 * row * (copied + moved) + tables + 16 * len(add), "flops": 0}
    _, n = _ragged(case)
    words = (case["draft"] + 31) // 32
    return {"bytes": sum(n) * (4 + 12 + 4 * words) + case["batch"] * 8, "flops": 0}


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(shape, dtype, g):
    return torch.randn(shape, dtype=torch.float32 if math.prod(shape) < (1 << 24) else dtype, device="cuda", generator=g).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _pool(case, layers, pages, g):
    """K or V of a pool, seen as [layer, page, slot, head, dimension] whatever its order in memory."""
    dt, k, d, ps = DTYPES[case["dtype"]], case["n_kv"], case["dim"], case["page"]
    if case["layout"] == "slot":
        return _randn((layers, pages, ps, k, d), dt, g)
    return _randn((layers, pages, k, ps, d), dt, g).transpose(2, 3)


def _tables(need, spare, rng, extra=0):
    """Block tables over shuffled pages: need[b] pages for sequence b; unused entries are -1."""
    total = sum(need)
    perm = rng.permutation(total + spare)
    blocks = np.full((len(need), max(need) + extra), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        blocks[b, :n] = perm[at:at + n]
        at += n
    return blocks, total + spare


def _parents(n, rng):
    """A drafted tree: every node hangs on a recent one, now and then on the last committed token."""
    i = np.arange(n)
    p = i - 1 - np.minimum(rng.geometric(0.45, n) - 1, i)
    p[rng.random(n) < 0.05] = -1
    return p.astype(np.int32)


def _bits(parents, words):
    m = np.zeros((len(parents), words), np.uint32)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i // 32] |= np.uint32(1 << (i % 32))
    return m


def prepare(case, seed):
    g, rng, op = _gen(seed), np.random.default_rng(seed), case["op"]
    s = {"case": case, "op": op}
    if op in ("attn", "plan"):
        ctx, n = _ragged(case)
        cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        rows, words = int(cu[-1]), (case["draft"] + 31) // 32
        parents = [_parents(k, rng) for k in n]
        s.update(rows=rows, pad=case["pad"], words=words, cu=_ints(cu), most=max(n))
        s["len"] = _ints([c + k for c, k in zip(ctx, n)])
        if op == "plan":
            s["parent"] = _ints(np.concatenate(parents + [np.zeros(case["pad"], np.int32)]))
            for name, width in (("seq", 1), ("slot", 1), ("pos", 1), ("mask", words)):
                s[name] = torch.full((rows + case["pad"], width) if name == "mask" else (rows + case["pad"],), 7, dtype=torch.int32, device="cuda")
            s["fault"] = torch.zeros(1, dtype=torch.int32, device="cuda")
            return s
        mask = np.concatenate([_bits(p, words) for p in parents] + [np.zeros((case["pad"], words), np.uint32)])
        mask[rng.random(rows + case["pad"]) < 0.02] = 0  # nodes cut from their tree see the committed tokens alone, or nothing
        s["mask"] = torch.from_numpy(mask.view(np.int32)).cuda()
        blocks, pages = _tables([-(-(c + k) // case["page"]) for c, k in zip(ctx, n)], 3, rng)
        s["blocks"] = _ints(blocks)
        s["k"], s["v"] = _pool(case, 1, pages, g), _pool(case, 1, pages, g)
        q = (rows + case["pad"], case["n_head"], case["dim"])
        # scores of standard deviation 2: some keys stand out, as a trained model's do
        s["q"], s["out"] = _randn(q, DTYPES[case["dtype"]], g) * 2, _randn(q, DTYPES[case["dtype"]], g) * 0.01
        return s
    if op == "rope":
        ctx, n = _rope_rows(case)
        h, k, d, rows = case["n_head"], case["n_kv"], case["dim"], case["rows"]
        blocks, pages = _tables([-(-(c + m) // case["page"]) for c, m in zip(ctx, n)], 2, rng)
        s["blocks"] = _ints(blocks)
        s["x"] = _randn((rows + case["pad"], (h + 2 * k) * d), DTYPES[case["x"]], g)
        slot = np.concatenate([c + np.arange(m) for c, m in zip(ctx, n)] + [np.zeros(case["pad"])]).astype(np.int32)
        s["slot"] = _ints(slot)
        s["seq"] = _ints(np.concatenate([np.full(m, b) for b, m in enumerate(n)] + [np.full(case["pad"], -1)]).astype(np.int32))
        s["pos"] = s["slot"].clone()
        angle = np.arange(int(slot.max()) + 1)[:, None] * 500000.0 ** (-np.arange(0, d, 2) / d)[None]
        s["rope"] = torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)).cuda()
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
        s["k"], s["v"] = _pool(case, 1, pages, g), _pool(case, 1, pages, g)
        s["q"] = _randn((rows + case["pad"], h, d), DTYPES[case["dtype"]], g)
        return s
    length, parent, add = _page_lengths(case)
    slots, ps = case["seqs"] + case["forks"], case["page"]
    most = -(-(max(length) + case["draft"]) // ps)
    need = [-(-n // ps) for n in length]
    new = sum(-(-a // ps) + 2 for a in add)
    blocks, pages = _tables(need, new, rng, most - max(need))
    refs = np.zeros(pages, np.int32)
    refs[blocks[blocks >= 0]] = 1
    blocks = np.concatenate([blocks, np.full((case["forks"], most), -1, np.int32)])
    # the tables of a pool in one piece of memory: blocks, lengths, reference counts, fault word
    s["start"] = _ints(np.concatenate([blocks.reshape(-1), length, np.zeros(case["forks"]), refs, [0]]).astype(np.int32))
    s["tables"] = s["start"].clone()
    s.update(slots=slots, max_blocks=most, pages=pages)
    s["src"], s["dst"] = _ints(parent), _ints(list(range(case["seqs"], slots)))
    s["all"], s["add"] = _ints(list(range(slots))), _ints(add)
    kept = [int(rng.integers(0, a + 1)) for a in add]
    path = np.zeros((slots, case["draft"]), np.int32)
    for i, (a, m) in enumerate(zip(add, kept)):
        path[i, :m] = np.sort(rng.choice(a, m, replace=False))
    s["path"], s["kept"] = _ints(path), _ints(kept)
    # every other fork loses and is released
    s["lost"] = _ints(list(range(case["seqs"], slots, 2)))
    s["k"], s["v"] = _pool(case, case["layers"], pages, g), _pool(case, case["layers"], pages, g)
    return s


# ---------------------------------------------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------------------------------------------
_context = {}


def _lib():
    from ullm_b200 import backend

    dev = torch.cuda.current_device()
    if dev not in _context:
        _context[dev] = backend.CudaContext(dev)
    return backend, _context[dev]


def _stream():
    # the library takes a null stream as the context's own; cudaStreamLegacy (1) names torch's default stream
    return torch.cuda.current_stream().cuda_stream or 1


def _pages(backend, s):
    case, st = s["case"], s["k"].stride()
    ids = {"f32": backend.F32, "f16": backend.F16, "bf16": backend.BF16}
    return backend.KvPages(ids[case["dtype"]], s["k"].shape[0], s["k"].shape[1], case["page"], case["n_kv"], case["dim"], s["k"].data_ptr(),
                           s["v"].data_ptr(), strides=st[:4])


def _own_attn(s):
    case = s["case"]
    if "call" not in s:
        backend, ctx = _lib()
        s["call"] = backend.TreeAttention(ctx, _pages(backend, s), case["n_head"])
    s["call"].run_dev(0, s["q"].data_ptr(), s["out"].data_ptr(), s["rows"] + s["pad"], case["batch"], s["cu"].data_ptr(), s["len"].data_ptr(),
                      s["blocks"].data_ptr(), s["blocks"].shape[1], d_mask=s["mask"].data_ptr(), mask_words=s["words"], stream=_stream())
    return s["out"]


def _own_plan(s):
    _, ctx = _lib()
    ctx.tree_plan_dev(s["rows"] + s["pad"], s["case"]["batch"], s["cu"].data_ptr(), s["len"].data_ptr(), s["parent"].data_ptr(), s["seq"].data_ptr(),
                      s["slot"].data_ptr(), s["pos"].data_ptr(), s["mask"].data_ptr(), s["words"], s["fault"].data_ptr(), stream=_stream())
    return [s["seq"], s["slot"], s["pos"], s["mask"]]


def _own_rope(s):
    case = s["case"]
    h, k, d = case["n_head"], case["n_kv"], case["dim"]
    if "call" not in s:
        backend, ctx = _lib()
        x = {"f32": backend.F32, "f16": backend.F16, "bf16": backend.BF16}[case["x"]]
        s["call"] = backend.QkNormRope(ctx, _pages(backend, s), h, x_dtype=x, d_rope=s["rope"].data_ptr(), n_pos=s["rope"].shape[0], neox=case["neox"],
                                       d_q_norm=s["q_norm"].data_ptr() if case["norm"] else None,
                                       d_k_norm=s["k_norm"].data_ptr() if case["norm"] else None, eps=1e-6)
    p, w, e = s["x"].data_ptr(), (h + 2 * k) * d, s["x"].element_size()
    s["call"].run_dev(0, p, p + h * d * e, p + (h + k) * d * e, s["q"].data_ptr(), s["x"].shape[0], s["pos"].data_ptr(), s["seq"].data_ptr(),
                      s["slot"].data_ptr(), s["blocks"].data_ptr(), s["blocks"].shape[0], s["blocks"].shape[1], x_stride=w, stream=_stream())
    return [s["q"], s["k"], s["v"]]


def _split(s):
    t, a, b = s["tables"], s["slots"] * s["max_blocks"], s["slots"]
    return t[:a].view(s["slots"], s["max_blocks"]), t[a:a + b], t[a + b:a + b + s["pages"]], t[a + b + s["pages"]:]


def _own_pages(s):
    case, st = s["case"], _stream()
    s["tables"].copy_(s["start"])
    blocks, length, refs, fault = _split(s)
    if "call" not in s:
        backend, ctx = _lib()
        s["call"] = backend.KvTable(ctx, _pages(backend, s), blocks.data_ptr(), length.data_ptr(), refs.data_ptr(), fault.data_ptr(), s["slots"],
                                    s["max_blocks"])
    t = s["call"]
    if case["forks"]:
        t.fork_dev(s["src"].data_ptr(), s["dst"].data_ptr(), case["forks"], stream=st)
    t.grow_dev(s["all"].data_ptr(), s["add"].data_ptr(), s["slots"], stream=st)
    t.accept_dev(s["all"].data_ptr(), s["add"].data_ptr(), s["path"].data_ptr(), s["kept"].data_ptr(), s["slots"], s["path"].shape[1], stream=st)
    if case["forks"]:
        t.trim_dev(s["lost"].data_ptr(), None, s["lost"].shape[0], stream=st)
    return [blocks, length, refs, fault, s["k"], s["v"]]


# ---------------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------------
def _plain_attn(s):
    case = s["case"]
    b, h, k, d, ps = case["batch"], case["n_head"], case["n_kv"], case["dim"], case["page"]
    rows, n, g = s["rows"], s["most"], case["n_head"] // case["n_kv"]
    page = s["blocks"].clamp(min=0).long()
    keys = s["k"][0][page].reshape(b, -1, k, d).float().permute(0, 2, 3, 1)    # [b, k, d, keys]
    vals = s["v"][0][page].reshape(b, -1, k, d).float().permute(0, 2, 1, 3)    # [b, k, keys, d]
    cu, length = s["cu"].long(), s["len"].long()
    count = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + torch.arange(n, device="cuda")).clamp(max=rows - 1)   # [b, n]: the padded batch's rows
    q = s["q"][at].float().view(b, n, k, g, d).permute(0, 2, 1, 3, 4).reshape(b, k, n * g, d)
    score = torch.matmul(q, keys).view(b, k, n, g, -1) * (1.0 / math.sqrt(d))
    key = torch.arange(ps * page.shape[1], device="cuda")
    node = key[None] - (length - count)[:, None]                                # [b, keys]: index among the drafted tokens
    word = (node.clamp(min=0) // 32).clamp(max=s["words"] - 1)
    bits = torch.gather(s["mask"][at], 2, word[:, None].expand(b, n, -1)) >> (node.clamp(min=0) % 32).int()[:, None]
    seen = ((node < 0)[:, None] | ((bits & 1) == 1)) & (key[None, None] < length[:, None, None])
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(b, k, n * g, -1), vals).view(b, k, n, g, d) / torch.where(total == 0, torch.ones_like(total), total)
    row = torch.arange(rows, device="cuda")
    seq = torch.bucketize(row, cu[1:], right=True)
    s["out"][:rows] = out.permute(0, 2, 1, 3, 4).reshape(b, n, h, d)[seq, row - cu[seq]].to(s["out"].dtype)
    return s["out"]


def _plain_plan(s):
    rows, n, words, cu = s["rows"], s["most"], s["words"], s["cu"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.bucketize(row, cu[1:], right=True)
    me = row - cu[seq]
    par = s["parent"][:rows].long()
    # ancestors by doubling: `sees` holds a node's ancestors up to 2^i steps away, itself among them, and `jump` the 2^i-th
    sees = torch.zeros(rows, n + 1, dtype=torch.bool, device="cuda")
    sees[row, me] = True
    jump = torch.where(par >= 0, cu[seq] + par, rows)
    none = torch.zeros(1, n + 1, dtype=torch.bool, device="cuda")
    for _ in range(max(1, (n - 1).bit_length())):
        sees = sees | torch.cat([sees, none])[jump]
        jump = torch.cat([jump, jump.new_full((1,), rows)])[jump]
    sees = sees[:, :n]
    count = cu[1:] - cu[:-1]
    first = (s["len"].long() - count)[seq]
    s["seq"][:rows], s["slot"][:rows] = seq.int(), (first + me).int()
    s["pos"][:rows] = (first + sees.sum(1) - 1).int()
    bits = torch.zeros(rows, words * 32, dtype=torch.int64, device="cuda")
    bits[:, :n] = sees
    value = (bits.view(rows, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    s["mask"][:rows] = torch.where(value >= 1 << 31, value - (1 << 32), value).int()
    s["seq"][rows:] = -1
    return [s["seq"], s["slot"], s["pos"], s["mask"]]


def _plain_rope(s):
    case = s["case"]
    h, k, d, ps, rows = case["n_head"], case["n_kv"], case["dim"], case["page"], case["rows"]
    x = s["x"][:rows].float()
    q, key, val = x[:, :h * d].view(rows, h, d), x[:, h * d:(h + k) * d].view(rows, k, d), x[:, (h + k) * d:].view(rows, k, d)
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_norm"]
        key = key * torch.rsqrt(key.square().mean(-1, keepdim=True) + 1e-6) * s["k_norm"]
    cs = s["rope"][s["pos"][:rows].long()]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]

    def turn(t):
        a, b = (t[..., :d // 2], t[..., d // 2:]) if case["neox"] else (t[..., 0::2], t[..., 1::2])
        u, w = a * cos - b * sin, a * sin + b * cos
        return torch.cat([u, w], -1) if case["neox"] else torch.stack([u, w], -1).flatten(-2)

    dt = DTYPES[case["dtype"]]
    s["q"][:rows] = turn(q).to(dt)
    slot = s["slot"][:rows].long()
    page = s["blocks"][s["seq"][:rows].long(), slot // ps].long()
    s["k"][0, page, slot % ps] = turn(key).to(dt)
    s["v"][0, page, slot % ps] = val.to(dt)
    return [s["q"], s["k"], s["v"]]


def _plain_pages(s):
    case, ps, mb = s["case"], s["case"]["page"], s["max_blocks"]
    s["tables"].copy_(s["start"])
    blocks, length, refs, fault = _split(s)
    col = torch.arange(mb, device="cuda")

    def held(seq):
        """Which entries of these sequences' tables are in use, and the pages there."""
        return col[None] < ((length[seq] + ps - 1) // ps)[:, None], blocks[seq].long()

    if case["forks"]:  # share: the child takes the parent's pages
        src, dst = s["src"].long(), s["dst"].long()
        use, page = held(src)
        blocks[dst] = torch.where(use, blocks[src], blocks[dst])
        length[dst] = length[src]
        refs.index_add_(0, page[use], torch.ones_like(page[use], dtype=torch.int32))
    # grow: pages for the new tokens, the lowest free ones first; a shared page that will be written is copied
    seq, add, n = s["all"].long(), s["add"].long(), s["slots"]
    old = length.long()
    part = old % ps
    last = (old // ps).clamp(max=mb - 1)
    cow = (part > 0) & (refs[blocks[seq, last].clamp(min=0).long()] > 1)
    have, want = (old + ps - 1) // ps, (old + add + ps - 1) // ps
    need = want - have + cow
    free = torch.nonzero(refs == 0)[:, 0]
    start = torch.cumsum(need, 0) - need
    took = (col[None] >= (have - cow.long())[:, None]) & (col[None] < want[:, None])
    pick = (start[:, None] + col[None] - (have - cow.long())[:, None])[took]
    before, after = blocks[seq, last].long()[cow], free[start[cow]]
    blocks[took] = free[pick].int()
    refs[free[pick]] = 1
    refs.index_add_(0, before, -torch.ones_like(before, dtype=torch.int32))
    inside = torch.arange(ps, device="cuda")[None] < part[cow][:, None]
    who, slot = torch.nonzero(inside, as_tuple=True)
    for pool in (s["k"], s["v"]):
        pool[:, after[who], slot] = pool[:, before[who], slot]
    length.add_(s["add"])
    # accept: the kept rows of every draft move up behind the committed tokens
    path, kept = s["path"].long(), s["kept"].long()
    j = torch.arange(path.shape[1], device="cuda")
    who, j = torch.nonzero(j[None] < kept[:, None], as_tuple=True)
    at, to = (old[who] + path[who, j]), old[who] + j
    src, dst = blocks[who, at // ps].long(), blocks[who, to // ps].long()
    for pool in (s["k"], s["v"]):
        pool[:, dst, to % ps] = pool[:, src, at % ps].clone()
    now = old + kept

    def cut(seq, new):  # free the pages behind the new lengths
        use, page = held(seq)
        gone = use & (col[None] >= ((new + ps - 1) // ps)[:, None])
        refs.index_add_(0, page[gone], -torch.ones_like(page[gone], dtype=torch.int32))
        length[seq] = new.int()

    cut(seq, now)
    if case["forks"]:
        cut(s["lost"].long(), torch.zeros_like(s["lost"]).long())
    return [blocks, length, refs, fault, s["k"], s["v"]]


def run(state):
    if own:
        return {"attn": _own_attn, "plan": _own_plan, "rope": _own_rope, "pages": _own_pages}[state["op"]](state)
    return {"attn": _plain_attn, "plan": _plain_plan, "rope": _plain_rope, "pages": _plain_pages}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------
# In 64 bits, sequence by sequence and row by row, from the definitions
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] not in ("attn", "rope"):
        return None
    s = prepare(case, seed)
    ps, h, k, d = case["page"], case["n_head"], case["n_kv"], case["dim"]
    blocks = s["blocks"].cpu().numpy()
    if case["op"] == "attn":
        out = s["out"].double()
        cu, length = s["cu"].tolist(), s["len"].tolist()
        mask = s["mask"].cpu().numpy().view(np.uint32)
        for b in range(case["batch"]):
            n, total = cu[b + 1] - cu[b], length[b]
            token = np.arange(total)
            page, slot = torch.from_numpy(blocks[b, token // ps].astype(np.int64)).cuda(), torch.from_numpy(token % ps).cuda()
            see = np.ones((n, total), bool)
            for i in range(n):
                for j in range(n):
                    see[i, total - n + j] = (int(mask[cu[b] + i, j // 32]) >> (j % 32)) & 1
            see = torch.from_numpy(see).cuda()
            for kv in range(k):
                key, val = s["k"][0, page, slot, kv].double(), s["v"][0, page, slot, kv].double()
                for head in range(kv * (h // k), (kv + 1) * (h // k)):
                    a = s["q"][cu[b]:cu[b + 1], head].double() @ key.T / math.sqrt(d)
                    a = torch.where(see, a, torch.full_like(a, -math.inf))
                    out[cu[b]:cu[b + 1], head] = torch.nan_to_num(torch.softmax(a, -1), nan=0.0) @ val
        return out
    rows = case["rows"]
    q_out, k_out, v_out = s["q"].double(), s["k"].double(), s["v"].double()
    slot = s["slot"].cpu().numpy()[:rows]
    page = torch.from_numpy(blocks[s["seq"].cpu().numpy()[:rows], slot // ps].astype(np.int64)).cuda()
    where = torch.from_numpy((slot % ps).astype(np.int64)).cuda()
    turn = torch.view_as_complex(s["rope"].double().contiguous())[s["pos"][:rows].long()]
    for head in range(h + 2 * k):
        t = s["x"][:rows, head * d:(head + 1) * d].double()
        if head >= h + k:
            v_out[0, page, where, head - h - k] = t
            continue
        if case["norm"]:
            t = t / torch.sqrt((t * t).sum(-1, keepdim=True) / d + 1e-6) * (s["q_norm"] if head < h else s["k_norm"]).double()
        i = torch.arange(d // 2, device="cuda")
        first, second = (i, i + d // 2) if case["neox"] else (2 * i, 2 * i + 1)
        z = torch.complex(t[:, first], t[:, second]) * turn
        r = torch.empty_like(t)
        r[:, first], r[:, second] = z.real, z.imag
        if head < h:
            q_out[:rows, head] = r
        else:
            k_out[0, page, where, head - h] = r
    return [q_out, k_out, v_out]
