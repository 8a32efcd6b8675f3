"""GPU tests of a tree of drafted tokens through the resident engine (``ullm_cuda_forward_verify`` / ``_accept``): every node's logits
against the engine's own decode step run along the node's path, with an f32 cache against the oracle's ``forward_llama`` too
(crates/ullm-model/src/lib.rs:807-969), and decoding that goes on from the accepted tokens.

The oracle's bar is not asked of an f16 cache: the decode step's projections are 3e-5 from the oracle's, so that a key now and then rounds
to the neighbouring f16 value, and where two keys of these random models nearly tie the logits then move by more than the bar - the
decode step's own (3.7e-3 at one node of this tree) by exactly what the tree's do."""
import numpy as np
import pytest

import oracle
import paged_ref
import test_moe_forward_gpu
import test_prefill_gpu
from test_decode_gpu import variant_model
from ullm_b200 import backend, synth

pytestmark = pytest.mark.gpu
TOL = 1e-3       # the bar of the decode step (its matvecs)
# Against the decode step itself.  Where norms of heads or attention sum in another order their results differ in the last bit (2^-23); a matvec re-expresses its
# input as 16-bit fixed point, so that such a difference now and then moves an element by a whole step (2^-16 of its group's largest):
# an error of the size, and with the bound, of what the matvec differs from the f32 product by anyway, 3e-5 each and 1e-3 for a whole
# step.  Without norms nothing differs and the chain test below asks for 1e-4.
SAME = 1e-3
TOL_BF16 = 2e-2  # the bar of products with bf16 operands


def build(ctx, kind, kv_f16):
    """(oracle model, engine) of a small model."""
    if kind == "moe":
        m = synth.gen_qwen3moe_model(dict(synth.QWEN3MOE_TINY), 3)
        return test_moe_forward_gpu.oracle_model(m, kv_f16), backend.GpuForward(ctx, m, kv_f16=kv_f16, rope_neox=1, qk_norm=1)
    bias, norm, neox = kind in ("bias", "all"), kind in ("norm", "all"), kind in ("neox", "all")
    m = variant_model(dict(synth.LLAMA_TINY), 31, bias, norm)
    mk = lambda t: oracle.Weight(t[0], t[1], t[2], t[3])  # noqa: E731
    layers = [{k: (mk(v) if isinstance(v, tuple) else v) for k, v in l.items()} for l in m["layers"]]
    om = oracle.LlamaModel(m["params"], mk(m["tok_embd"]), mk(m["output"]), m["final_norm"], layers, kv_f16, rope_neox=neox)
    return om, backend.GpuForward(ctx, m, kv_f16=kv_f16, rope_neox=1 if neox else 0, qk_norm=1 if norm else 0)


def path_to(parents, i):
    p = []
    while i >= 0:
        p.insert(0, i)
        i = int(parents[i])
    return p


@pytest.mark.parametrize("kind,kv_f16", [("plain", False), ("plain", True), ("bias", True), ("norm", False), ("all", True), ("moe", False), ("moe", True)])
def test_every_node_sees_its_own_path_and_decoding_goes_on(ctx, kind, kv_f16):
    om, gf = build(ctx, kind, kv_f16)
    _, step = build(ctx, kind, kv_f16)
    rng = np.random.default_rng(5)
    prompt = [7, 30, 12, 99, 4]
    for pos, tok in enumerate(prompt):
        gf.forward(om.embed(tok), pos)
    committed = list(prompt)

    def check(got, tokens):
        """`got` against the logits of the last of these tokens, each decoded at its position."""
        assert synth.rel_err(got, [step.forward(om.embed(t), i) for i, t in enumerate(tokens)][-1]) < SAME
        if not kv_f16:
            assert synth.rel_err(got, [om.forward(t, i) for i, t in enumerate(tokens)][-1]) < TOL

    for n, keep in ((1, 0), (6, 3), (11, 10), (3, 1)):
        parents = paged_ref.tree_parents(n, rng, 0.3)
        tokens = [int(t) for t in rng.integers(0, 200, n)]
        got = gf.verify(np.stack([om.embed(t) for t in tokens]), len(committed), parents)
        for i in range(n):
            check(got[i], committed + [tokens[j] for j in path_to(parents, i)])
        path = path_to(parents, keep)
        gf.accept(len(committed), n, path)
        committed += [tokens[j] for j in path]
        tok = int(rng.integers(0, 200))
        check(gf.forward(om.embed(tok), len(committed)), committed + [tok])
        committed.append(tok)
    # nothing accepted: the next token overwrites the first draft
    gf.verify(np.stack([om.embed(t) for t in (1, 2, 3)]), len(committed))
    gf.accept(len(committed), 3, [])
    check(gf.forward(om.embed(50), len(committed)), committed + [50])
    gf.free(), step.free()


@pytest.mark.parametrize("kv_f16", [False, True])
def test_a_chain_gives_the_decode_steps_logits(ctx, kv_f16):
    om, a = build(ctx, "plain", kv_f16)
    _, b = build(ctx, "plain", kv_f16)
    tokens = [5, 80, 33, 2, 150, 61, 9]
    step = [a.forward(om.embed(t), i) for i, t in enumerate(tokens)]
    got = b.verify(np.stack([om.embed(t) for t in tokens]), 0)
    for i in range(len(tokens)):  # the same matvecs; the two attentions differ in the order of their f32 sums
        assert synth.rel_err(got[i], step[i]) < 1e-4 and int(np.argmax(got[i])) == int(np.argmax(step[i]))
    assert synth.rel_err(b.forward(om.embed(3), 7), a.forward(om.embed(3), 7)) < 1e-4
    a.free(), b.free()


def test_more_tokens_run_on_the_tensor_cores(ctx):
    p = dict(test_prefill_gpu.SMALL)
    m = test_prefill_gpu.conditioned(synth.gen_llama_model(p, 9))
    om = test_prefill_gpu.oracle_model(m, True)
    gf = backend.GpuForward(ctx, m, kv_f16=True)
    assert gf.supports_batched_prefill()
    rng = np.random.default_rng(2)
    prompt = [int(t) for t in rng.integers(0, p["vocab"], 40)]
    gf.forward_batch(np.stack([om.embed(t) for t in prompt]), len(prompt))
    for n in (8, 33, 64):
        parents = paged_ref.tree_parents(n, rng, 0.2)
        tokens = [int(t) for t in rng.integers(0, p["vocab"], n)]
        got = gf.verify(np.stack([om.embed(t) for t in tokens]), len(prompt), parents)
        for i in (0, n // 2, n - 1):
            seq = prompt + [tokens[j] for j in path_to(parents, i)]
            ref = test_prefill_gpu.prefill_reference(m, np.stack([om.embed(t) for t in seq]), True, True)
            assert synth.rel_err(got[i], ref) < TOL_BF16, (n, i)
    gf.free()


def test_refusals(ctx):
    om, gf = build(ctx, "plain", False)
    e = np.stack([om.embed(t) for t in range(65)])
    for call in (lambda: gf.verify(e, 0), lambda: gf.verify(e[:0], 0), lambda: gf.verify(e[:4], 61), lambda: gf.verify(e[:4], 1 << 40), lambda: gf.verify(e[:3], 0, [-1, 1, 0]),
                 lambda: gf.verify(e[:3], 0, [0, 0, 0]), lambda: gf.verify(e[:3], 0, [-2, 0, 0]), lambda: gf.accept(0, 3, [0, 0]), lambda: gf.accept(0, 3, [2, 1]),
                 lambda: gf.accept(0, 3, [-1]), lambda: gf.accept(0, 3, [1, 3]), lambda: gf.accept(0, 0, []), lambda: gf.accept(62, 3, [0]), lambda: gf.accept(0, 65, [0])):
        with pytest.raises(backend.FormatError):
            call()
    lib = backend.load_library()
    assert lib.ullm_cuda_forward_verify(None, None, None, 1, 0, None) == backend.ERR_INVALID
    assert lib.ullm_cuda_forward_accept(gf._h, 0, 3, None, 1) == backend.ERR_INVALID
    gf.verify(e[:4], 60)  # the last four positions
    gf.free()


@pytest.mark.parametrize("kv_f16,n", [(False, 6), (True, 6), (False, 1)])
def test_a_tree_behind_a_long_context(ctx, kv_f16, n):
    """Two thousand cached positions: the attention's units are cut into parts."""
    p = dict(synth.LLAMA_TINY, n_ctx=2100)
    m = variant_model(p, 31, False, False)
    a, b = backend.GpuForward(ctx, m, kv_f16=kv_f16), backend.GpuForward(ctx, m, kv_f16=kv_f16)
    rng = np.random.default_rng(8)
    pos, width = 2000, p["n_kv_head"] * p["head_dim"]
    k, v = (rng.standard_normal((p["n_layer"], pos, width)).astype(np.float32) for _ in range(2))
    e = rng.standard_normal((n, p["n_embd"])).astype(np.float32)
    parents = paged_ref.tree_parents(n, rng, 0.3)
    for f in (a, b):
        f.set_kv(0, k, v)
    got = a.verify(e, pos, parents)
    for i in range(n):
        path = path_to(parents, i)
        assert synth.rel_err(got[i], [b.forward(e[j], pos + d) for d, j in enumerate(path)][-1]) < SAME
    path = path_to(parents, n - 1)
    a.accept(pos, n, path)
    x = rng.standard_normal(p["n_embd"]).astype(np.float32)
    assert synth.rel_err(a.forward(x, pos + len(path)), b.forward(x, pos + len(path))) < SAME
    a.free(), b.free()
