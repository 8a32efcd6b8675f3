"""CPU tests of the paged-cache operators' boundary: what the host refuses before anything is launched, and the
reference rules themselves on small cases."""
import ctypes as C

import numpy as np
import pytest

import paged_ref
from ullm_b200 import backend

LIB = backend.load_library()
# A context of zero bytes: enough for the checks of arguments, which come before the first CUDA call.  A call that
# passed them would end with a CUDA error here (there is no device), not with the codes asserted below.
FAKE = C.create_string_buffer(1 << 14)
CTX = C.addressof(FAKE)
P = 1 << 20  # an aligned address that nothing reads


def pages(**kw):
    a = dict(dtype=backend.F16, n_layer=2, n_pages=10, page_size=16, n_kv_head=2, head_dim=64, d_k=P, d_v=P)
    strides = kw.pop("strides", None)
    a.update(kw)
    return backend.KvPages(**a, strides=strides)


def table(kv, **kw):
    a = dict(d_blocks=P, d_len=P, d_refs=P, d_fault=P, n_seq=4, max_blocks=8, d_work=P)
    a.update(kw)
    a.setdefault("work_bytes", LIB.ullm_cuda_kv_work_bytes(kv.n_pages, a["n_seq"]))
    return backend.KvTableC(*[a[n] for n, _ in backend.KvTableC._fields_])


BAD_POOLS = [
    (dict(dtype=backend.Q4_K), backend.ERR_FORMAT), (dict(n_layer=0), backend.ERR_FORMAT), (dict(n_pages=0), backend.ERR_FORMAT),
    (dict(page_size=0), backend.ERR_FORMAT), (dict(n_kv_head=0), backend.ERR_FORMAT), (dict(head_dim=0), backend.ERR_FORMAT),
    (dict(head_dim=60), backend.ERR_FORMAT), (dict(head_dim=264), backend.ERR_FORMAT), (dict(d_k=P + 8), backend.ERR_FORMAT),
    (dict(d_k=None), backend.ERR_INVALID), (dict(d_v=None), backend.ERR_INVALID), (dict(n_pages=1 << 31), backend.ERR_FORMAT),
    (dict(page_size=1 << 20), backend.ERR_FORMAT), (dict(strides=(4096 * 10, 4096, 130, 64)), backend.ERR_FORMAT),
    (dict(strides=(4096 * 10, 4096, 128, 32)), backend.ERR_FORMAT),
]


@pytest.mark.parametrize("change,code", BAD_POOLS)
def test_every_call_refuses_a_bad_pool(change, code):
    kv = pages(**change)
    t = table(pages())
    t.work_bytes = 1 << 30
    k, tt = C.byref(kv), C.byref(t)
    assert LIB.ullm_cuda_kv_fork_dev(CTX, k, tt, P, P, 1, None) == code
    assert LIB.ullm_cuda_kv_grow_dev(CTX, k, tt, P, P, 1, None) == code
    assert LIB.ullm_cuda_kv_accept_dev(CTX, k, tt, P, P, P, P, 1, 4, None) == code
    assert LIB.ullm_cuda_kv_trim_dev(CTX, k, tt, P, None, 1, None) == code
    assert LIB.ullm_cuda_kv_copy_pages_dev(CTX, k, P, P, 1, None, None) == code
    r, a = rope(kv=C.addressof(kv)), attn(kv=C.addressof(kv))
    assert LIB.ullm_cuda_qk_norm_rope_dev(CTX, C.byref(r), None) == code
    assert LIB.ullm_cuda_tree_attn_dev(CTX, C.byref(a), None) in (code, backend.ERR_UNSUPPORTED if "dtype" in change else code)
    if code == backend.ERR_FORMAT:
        assert LIB.ullm_cuda_tree_attn_work_bytes(CTX, k, backend.F16) == 0


@pytest.mark.parametrize("change,code", [
    (dict(d_blocks=None), backend.ERR_INVALID), (dict(d_len=None), backend.ERR_INVALID), (dict(d_refs=None), backend.ERR_INVALID),
    (dict(d_fault=None), backend.ERR_INVALID), (dict(d_work=None), backend.ERR_INVALID), (dict(n_seq=0, work_bytes=1 << 20), backend.ERR_FORMAT),
    (dict(max_blocks=0), backend.ERR_FORMAT), (dict(max_blocks=1 << 27), backend.ERR_FORMAT), (dict(work_bytes=8), backend.ERR_FORMAT),
    (dict(d_len=P + 2), backend.ERR_FORMAT), (dict(n_seq=1), backend.ERR_FORMAT),
])
def test_tables_are_checked(change, code):
    kv = pages()
    t = table(kv, **change)
    k, tt = C.byref(kv), C.byref(t)
    assert LIB.ullm_cuda_kv_fork_dev(CTX, k, tt, P, P, 2, None) == code
    assert LIB.ullm_cuda_kv_grow_dev(CTX, k, tt, P, P, 2, None) == code
    assert LIB.ullm_cuda_kv_accept_dev(CTX, k, tt, P, P, P, P, 2, 4, None) == code
    assert LIB.ullm_cuda_kv_trim_dev(CTX, k, tt, P, None, 2, None) == code


def test_null_lists_and_contexts_and_empty_calls():
    kv = pages()
    t = table(kv)
    k, tt = C.byref(kv), C.byref(t)
    assert LIB.ullm_cuda_kv_fork_dev(None, k, tt, P, P, 1, None) == backend.ERR_INVALID
    assert LIB.ullm_cuda_kv_fork_dev(CTX, k, tt, None, P, 1, None) == backend.ERR_INVALID
    assert LIB.ullm_cuda_kv_grow_dev(CTX, k, tt, P, None, 1, None) == backend.ERR_INVALID
    assert LIB.ullm_cuda_kv_accept_dev(CTX, k, tt, P, P, None, P, 1, 4, None) == backend.ERR_INVALID
    assert LIB.ullm_cuda_kv_trim_dev(CTX, k, tt, None, None, 1, None) == backend.ERR_INVALID
    assert LIB.ullm_cuda_kv_trim_dev(CTX, None, tt, P, None, 1, None) == backend.ERR_INVALID
    assert LIB.ullm_cuda_kv_copy_pages_dev(CTX, k, P, P, 11, None, None) == backend.ERR_FORMAT  # more copies than pages
    assert LIB.ullm_cuda_kv_accept_dev(CTX, k, tt, P, P, P, P, 1, 1 << 40, None) == backend.ERR_FORMAT
    # nothing to do is no error and touches no device
    assert LIB.ullm_cuda_kv_fork_dev(CTX, k, tt, None, None, 0, None) == backend.OK
    assert LIB.ullm_cuda_kv_grow_dev(CTX, k, tt, None, None, 0, None) == backend.OK
    assert LIB.ullm_cuda_kv_accept_dev(CTX, k, tt, None, None, None, None, 0, 4, None) == backend.OK
    assert LIB.ullm_cuda_kv_trim_dev(CTX, k, tt, None, None, 0, None) == backend.OK
    assert LIB.ullm_cuda_kv_copy_pages_dev(CTX, k, None, None, 0, None, None) == backend.OK
    assert LIB.ullm_cuda_qk_norm_rope_dev(CTX, C.byref(rope(n_rows=0)), None) == backend.OK
    assert LIB.ullm_cuda_tree_attn_dev(CTX, C.byref(attn(n_rows=0)), None) == backend.OK
    assert LIB.ullm_cuda_tree_attn_dev(CTX, C.byref(attn(n_seq=0)), None) == backend.OK


KEEP = []


def rope(**kw):
    kv = pages()
    KEEP.append(kv)
    a = dict(kv=C.addressof(kv), layer=1, x_dtype=backend.F32, q_dtype=backend.F16, n_rows=3, n_head=4, d_q=P, d_k=P, d_v=P, q_stride=0, k_stride=0, v_stride=0,
             d_q_out=P, q_out_stride=0, d_q_norm=P, d_k_norm=P, d_q_bias=None, d_k_bias=None, d_v_bias=None, eps=1e-6, d_rope=P, n_pos=8, rot_dim=0, neox=0,
             d_row_seq=P, d_row_slot=P, d_row_pos=P, d_blocks=P, n_table=2, max_blocks=4, d_fault=None)
    a.update(kw)
    return backend.QkNormRopeC(*[a[n] for n, _ in backend.QkNormRopeC._fields_])


@pytest.mark.parametrize("change,code", [
    (dict(kv=None), backend.ERR_INVALID), (dict(d_q=None), backend.ERR_INVALID), (dict(d_k=None), backend.ERR_INVALID), (dict(d_v=None), backend.ERR_INVALID),
    (dict(d_q_out=None), backend.ERR_INVALID), (dict(d_rope=None), backend.ERR_INVALID), (dict(d_row_seq=None), backend.ERR_INVALID),
    (dict(d_row_slot=None), backend.ERR_INVALID), (dict(d_row_pos=None), backend.ERR_INVALID), (dict(d_blocks=None), backend.ERR_INVALID),
    (dict(x_dtype=backend.Q4_K), backend.ERR_UNSUPPORTED), (dict(q_dtype=backend.BF16), backend.ERR_UNSUPPORTED), (dict(layer=2), backend.ERR_FORMAT),
    (dict(n_head=0), backend.ERR_FORMAT), (dict(rot_dim=24), backend.ERR_FORMAT), (dict(rot_dim=80), backend.ERR_FORMAT), (dict(d_k_norm=None), backend.ERR_FORMAT),
    (dict(n_pos=0), backend.ERR_FORMAT), (dict(n_table=0), backend.ERR_FORMAT), (dict(max_blocks=0), backend.ERR_FORMAT), (dict(q_stride=128), backend.ERR_FORMAT),
    (dict(k_stride=129), backend.ERR_FORMAT), (dict(q_out_stride=252), backend.ERR_FORMAT), (dict(d_q=P + 4), backend.ERR_FORMAT),
    (dict(d_v_bias=P + 4), backend.ERR_FORMAT), (dict(d_rope=P + 8), backend.ERR_FORMAT), (dict(n_rows=1 << 31), backend.ERR_FORMAT),
])
def test_rope_arguments_are_checked(change, code):
    assert LIB.ullm_cuda_qk_norm_rope_dev(CTX, C.byref(rope(**change)), None) == code
    assert LIB.ullm_cuda_qk_norm_rope_dev(None, C.byref(rope()), None) == backend.ERR_INVALID


def attn(**kw):
    kv = pages()
    KEEP.append(kv)
    a = dict(kv=C.addressof(kv), layer=1, dtype=backend.F16, n_rows=3, n_seq=2, n_head=4, d_q=P, q_stride=0, d_out=P, out_stride=0, d_cu=P, d_len=P, d_ids=None,
             d_blocks=P, n_table=2, max_blocks=4, d_mask=P, mask_words=1, scale=0.0, d_work=P, work_bytes=1 << 40)
    a.update(kw)
    return backend.TreeAttnC(*[a[n] for n, _ in backend.TreeAttnC._fields_])


@pytest.mark.parametrize("change,code", [
    (dict(kv=None), backend.ERR_INVALID), (dict(d_q=None), backend.ERR_INVALID), (dict(d_out=None), backend.ERR_INVALID), (dict(d_cu=None), backend.ERR_INVALID),
    (dict(d_len=None), backend.ERR_INVALID), (dict(d_blocks=None), backend.ERR_INVALID), (dict(d_work=None), backend.ERR_INVALID),
    (dict(dtype=backend.BF16), backend.ERR_UNSUPPORTED), (dict(layer=2), backend.ERR_FORMAT), (dict(n_head=3), backend.ERR_FORMAT),
    (dict(n_head=0), backend.ERR_FORMAT), (dict(n_table=1), backend.ERR_FORMAT), (dict(n_table=0), backend.ERR_FORMAT), (dict(max_blocks=0), backend.ERR_FORMAT),
    (dict(mask_words=0), backend.ERR_FORMAT), (dict(q_stride=192), backend.ERR_FORMAT), (dict(out_stride=260), backend.ERR_FORMAT),
    (dict(d_out=P + 8), backend.ERR_FORMAT), (dict(scale=float("nan")), backend.ERR_FORMAT), (dict(scale=-1.0), backend.ERR_FORMAT),
    (dict(d_work=P + 4), backend.ERR_FORMAT), (dict(n_rows=1 << 31), backend.ERR_FORMAT),
])
def test_attention_arguments_are_checked(change, code):
    assert LIB.ullm_cuda_tree_attn_dev(CTX, C.byref(attn(**change)), None) == code
    assert LIB.ullm_cuda_tree_attn_dev(None, C.byref(attn()), None) == backend.ERR_INVALID


@pytest.mark.parametrize("change,code", [
    (dict(cu=None), backend.ERR_INVALID), (dict(len=None), backend.ERR_INVALID), (dict(seq=None), backend.ERR_INVALID), (dict(pos=None), backend.ERR_INVALID),
    (dict(words=0), backend.ERR_FORMAT), (dict(words=1 << 20), backend.ERR_FORMAT), (dict(n_rows=1 << 31), backend.ERR_FORMAT), (dict(n_rows=0), backend.OK),
])
def test_plan_arguments_are_checked(change, code):
    a = dict(n_rows=4, n_seq=2, cu=P, len=P, ids=None, n_table=2, parent=P, seq=P, slot=P, pos=P, mask=P, words=1, fault=None)
    a.update(change)
    assert LIB.ullm_cuda_tree_plan_dev(CTX, *a.values(), None) == code


# ---- the reference rules on cases small enough to follow by hand ----
def small(n_seq=4, n_pages=8):
    k = np.arange(n_pages * 4, dtype=np.float64).reshape(1, n_pages, 4, 1, 1)
    return paged_ref.Tables(n_seq, 4, n_pages, 4, k.copy(), -k)


def test_reference_step_of_a_forked_sequence():
    t = small()
    t.grow([0], [6])
    assert t.blocks[0, :2].tolist() == [0, 1] and t.refs[:3].tolist() == [1, 1, 0]
    t.fork([0, 0], [1, 2])
    assert t.refs[:2].tolist() == [3, 3] and t.len[:3].tolist() == [6, 6, 6]
    t.grow([1, 0], [3, 0])  # row 1 writes into the shared second page: it gets a copy, then one more page
    assert t.blocks[1, :3].tolist() == [0, 2, 3] and t.refs[:4].tolist() == [3, 2, 1, 1]
    assert t.k[0, 2, :2, 0, 0].tolist() == [4, 5]
    t.accept([1], [3], np.array([[1, 2]]), [2])  # tokens 7 and 8 become 6 and 7; the last page is free again
    assert t.k[0, 2, 2:, 0, 0].tolist() == [11, 12] and t.len[1] == 8 and t.refs[3] == 0 and t.fault == 0
    t.trim([0, 2])
    t.trim([1], [0])
    assert t.refs.tolist() == [0] * 8 and t.fault == 0


def test_reference_refuses_bad_entries_and_keeps_the_others():
    t = small()
    t.grow([0, 1, 1, 9], [4, 1, 1, 1])
    assert t.fault == paged_ref.SEQ and t.len.tolist() == [4, 0, 0, 0]
    t.fault = 0
    t.grow([0, 2], [16, 2])  # row 0 would pass its four blocks
    assert t.fault == paged_ref.LEN and t.len.tolist() == [4, 0, 2, 0]
    t.fault = 0
    t.fork([0, 0, 2], [1, 1, 3])
    assert t.fault == paged_ref.SEQ and t.len.tolist() == [4, 0, 2, 2]
    t.fault = 0
    t.accept([3], [2], np.array([[1, 0]]), [2])
    assert t.fault == paged_ref.PATH | paged_ref.SHARED and t.len[3] == 2  # out of order, and into a page that row 2 shares
    t.fault = 0
    t.accept([3], [2], np.array([[1, 0]]), [1])
    assert t.fault == paged_ref.SHARED and t.len[3] == 2
    t.fault = 0
    t.grow([0, 1], [12, 16])  # seven pages are wanted, six are free
    assert t.fault == paged_ref.NO_PAGES and t.len.tolist() == [4, 0, 2, 2]


def test_reference_plan_of_a_small_tree():
    seq, slot, pos, mask, fault = paged_ref.plan([0, 4, 5], [10, 1], [-1, 0, 0, 2, -1], 7, words=1)
    assert seq.tolist() == [0, 0, 0, 0, 1, -1, -1] and slot[:5].tolist() == [6, 7, 8, 9, 0] and pos[:5].tolist() == [6, 7, 7, 8, 0]
    assert mask[:5, 0].tolist() == [0b1, 0b11, 0b101, 0b1101, 0b1] and fault == 0


class NoCalls:
    """A context whose library must not be reached."""

    def _check(self, code):
        raise AssertionError("called")

    def __getattr__(self, name):
        raise AssertionError(name)


@pytest.mark.parametrize("embeds,parents", [((3, 255), None), ((3, 257), None), ((256,), None), ((1, 3, 256), None), ((3, 256), [-1, 0]), ((3, 256), [-1, 0, 1, 2]), ((3, 256), []),
                                            ((3, 256), [[-1, 0, 1]])])
def test_verify_does_not_read_behind_its_arrays(embeds, parents):
    f = backend.GpuForward.__new__(backend.GpuForward)
    f._ctx, f._h, f.params = NoCalls(), None, dict(n_embd=256, vocab=8)
    with pytest.raises(backend.FormatError):
        f.verify(np.zeros(embeds, np.float32), 0, parents)


class Plain:
    """The library with a context that nothing is launched on (calls without rows)."""

    _lib, _h = LIB, CTX

    def _check(self, code):
        assert code == backend.OK


def test_a_layers_weights_are_given_with_its_calls():
    kv = pages()
    names = ("d_q_norm", "d_k_norm", "d_q_bias", "d_k_bias", "d_v_bias")
    op = backend.QkNormRope(Plain(), kv, 4, backend.F32, P, 8, d_q_norm=P, d_k_norm=P + 16, d_v_bias=P + 32)
    rows = dict(layer=0, d_q=P, d_k=P, d_v=P, d_q_out=P, n_rows=0, d_row_pos=P, d_row_seq=P, d_row_slot=P, d_blocks=P, n_table=2, max_blocks=4)
    for given in ({}, dict(d_q_norm=P + 64, d_k_norm=P + 80), dict(d_q_bias=P + 96, d_k_bias=P + 112, d_v_bias=P + 128), {}):
        op.run_dev(**rows, **given)
        assert [getattr(op._a, n) for n in names] == [given.get(n, w) for n, w in zip(names, (P, P + 16, None, None, P + 32))]


def test_lists_off_their_alignment_are_refused():
    """A 32-bit number off its boundary would end in a fault on the device."""
    kv = pages()
    t = table(kv)
    k, tt = C.byref(kv), C.byref(t)
    calls = [
        (lambda *p: LIB.ullm_cuda_kv_fork_dev(CTX, k, tt, *p, 1, None), 2), (lambda *p: LIB.ullm_cuda_kv_grow_dev(CTX, k, tt, *p, 1, None), 2),
        (lambda *p: LIB.ullm_cuda_kv_accept_dev(CTX, k, tt, *p, 1, 4, None), 4), (lambda *p: LIB.ullm_cuda_kv_trim_dev(CTX, k, tt, *p, 1, None), 2),
        (lambda s, d, f: LIB.ullm_cuda_kv_copy_pages_dev(CTX, k, s, d, 1, f, None), 3),
        (lambda cu, ln, ids, par, seq, slot, pos, mask, fault: LIB.ullm_cuda_tree_plan_dev(CTX, 4, 2, cu, ln, ids, 2, par, seq, slot, pos, mask, 1, fault, None), 9),
    ]
    for call, n in calls:
        for i in range(n):
            for off in (1, 2, 3):
                assert call(*[P + off if j == i else P for j in range(n)]) == backend.ERR_FORMAT
    for name in ("d_row_seq", "d_row_slot", "d_row_pos", "d_blocks", "d_fault"):
        assert LIB.ullm_cuda_qk_norm_rope_dev(CTX, C.byref(rope(**{name: P + 2})), None) == backend.ERR_FORMAT
    for name in ("d_cu", "d_len", "d_ids", "d_blocks", "d_mask"):
        assert LIB.ullm_cuda_tree_attn_dev(CTX, C.byref(attn(**{name: P + 2})), None) == backend.ERR_FORMAT


@pytest.mark.parametrize("scale", [2.5e38, 3.4e38, float("inf"), -float("inf"), 9e-31, -0.5])
def test_scales_that_are_no_number_in_powers_of_two_are_refused(scale):
    """The kernels work with scale * log2(e), which passes 32 bits from 2.36e38 on: every score of zero would become NaN."""
    assert LIB.ullm_cuda_tree_attn_dev(CTX, C.byref(attn(scale=scale)), None) == backend.ERR_FORMAT
