"""Refusals of the int8 LM head and the beam-search calls: checked before any GPU work, so they run
without one (pointers are placeholders that no kernel sees)."""
import ctypes as C

import pytest

from diskllm_b200 import capi

INVALID, UNSUPPORTED, OK = capi.DLLM_ERR_INVALID_ARG, capi.DLLM_ERR_UNSUPPORTED, capi.DLLM_OK
P = 4096  # an aligned placeholder


def _quantize(**kw):
    a = dict(rows=2, cols=20, x=P, x_stride=20, x_dtype=0, norm=0, norm_w=None, eps=1e-6, add_one=0, q=P, q_stride=32,
             scale=P)
    a.update(kw)
    return capi.load_library().dllm_cuda_quantize_rows_i8(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), OK), (dict(rows=0, x=None, q=None, scale=None), OK),
    (dict(rows=-1), INVALID), (dict(cols=0), INVALID), (dict(x_dtype=3), INVALID), (dict(x=None), INVALID),
    (dict(q=None), INVALID), (dict(scale=None), INVALID), (dict(x_stride=19), INVALID), (dict(q_stride=16), INVALID),
    (dict(q_stride=24), INVALID), (dict(q=P + 8), INVALID), (dict(x=P + 2), INVALID),
    (dict(x=P + 1, x_dtype=1), INVALID), (dict(norm_w=P), INVALID), (dict(add_one=1), INVALID),
    (dict(norm=1, eps=-1.0), INVALID), (dict(norm=1, eps=float("nan")), INVALID),
])
def test_quantize_refusals(kw, rc):
    assert _quantize(**kw) == rc
    if rc != OK:
        assert capi.load_library().dllm_cuda_last_error()


def _matmul(**kw):
    a = dict(m=2, n=3, k=20, a=P, lda=32, sa=P, b=P, ldb=32, sb=P, softcap=0.0, out=P, ldo=3, dtype=0, status=None)
    a.update(kw)
    return capi.load_library().dllm_cuda_matmul_i8(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(m=0), OK), (dict(n=0), OK), (dict(m=0, a=None, out=None), OK),
    (dict(m=-1), INVALID), (dict(n=-1), INVALID), (dict(k=0), INVALID), (dict(k=131072, lda=131072, ldb=131072), UNSUPPORTED),
    (dict(a=None), INVALID), (dict(b=None), INVALID), (dict(sa=None), INVALID), (dict(sb=None), INVALID),
    (dict(out=None), INVALID), (dict(lda=16), INVALID), (dict(lda=24), INVALID), (dict(ldb=24), INVALID),
    (dict(a=P + 4), INVALID), (dict(b=P + 1), INVALID), (dict(ldo=2), INVALID), (dict(dtype=5), INVALID),
    (dict(out=P + 2), INVALID), (dict(softcap=-1.0), INVALID), (dict(softcap=float("nan")), INVALID),
    (dict(softcap=float("inf")), INVALID),
])
def test_matmul_refusals(kw, rc):
    assert _matmul(**kw) == rc


def _lmhead(**kw):
    a = dict(rows=2, hidden=20, vocab=7, h=P, norm_w=None, eps=1e-6, add_one=0, w=P, ldw=32, sw=P, softcap=0.0, logits=P,
             status=None, ws=P, ws_bytes=1 << 20)
    a.update(kw)
    return capi.load_library().dllm_cuda_lmhead_logits_i8(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), OK), (dict(rows=-1), INVALID), (dict(hidden=0), INVALID), (dict(vocab=0), INVALID),
    (dict(h=None), INVALID), (dict(w=None), INVALID), (dict(sw=None), INVALID), (dict(logits=None), INVALID),
    (dict(ldw=16), INVALID), (dict(w=P + 8), INVALID), (dict(eps=-1.0), INVALID), (dict(softcap=-2.0), INVALID),
    (dict(ws=P + 16), INVALID), (dict(ws_bytes=64), INVALID), (dict(hidden=131072, ldw=131072), UNSUPPORTED),
])
def test_lmhead_refusals(kw, rc):
    assert _lmhead(**kw) == rc


def test_lmhead_workspace_bytes():
    f = capi.load_library().dllm_cuda_lmhead_i8_workspace_bytes
    assert f(0, 64) == 0 and f(3, 0) == 0
    assert f(1, 1) == 256 + 4        # one row of 16 bytes, rounded up, and its scale
    assert f(17, 100) == 2048 + 68   # 17 x 112


def _beam(**kw):
    d = capi.BeamDesc()
    a = dict(batch=2, beams=4, vocab=100, k=8, row_stride=100, dtype=0, logits=P, scores=P + 4096, eos=-1, out_score=P,
             out_parent=P, out_token=P, workspace=P, workspace_bytes=1 << 24)
    a.update(kw)
    for name, v in a.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("kw,rc", [
    (dict(batch=0), OK), (dict(batch=0, logits=None, scores=None), OK),
    (dict(batch=-1), INVALID), (dict(beams=0), INVALID), (dict(vocab=0), INVALID), (dict(k=0), INVALID),
    (dict(beams=129), UNSUPPORTED), (dict(k=257), UNSUPPORTED),
    (dict(vocab=2 ** 30 + 1, row_stride=2 ** 31), UNSUPPORTED), (dict(dtype=4), INVALID), (dict(row_stride=99), INVALID),
    (dict(logits=None), INVALID), (dict(scores=None), INVALID), (dict(out_score=None), INVALID),
    (dict(out_parent=None), INVALID), (dict(out_token=None), INVALID), (dict(logits=P + 2), INVALID),
    (dict(logits=P + 1, dtype=1), INVALID), (dict(mask=P, mask_stride=3), INVALID), (dict(finished=P), INVALID),
    (dict(out_finished=P), INVALID), (dict(length_penalty=1.0), INVALID), (dict(out_lengths=P), INVALID),
    (dict(length_penalty=float("nan"), lengths=P), INVALID), (dict(length_penalty=float("inf"), lengths=P), INVALID),
    (dict(workspace=P + 16), INVALID), (dict(workspace_bytes=16), INVALID),
    # outputs of another shape over the inputs: a sequence's would lie over the next one's inputs
    (dict(scores=P), INVALID), (dict(lengths=P, out_lengths=P), INVALID), (dict(eos=1, finished=P, out_finished=P), INVALID),
])
def test_beam_select_refusals(kw, rc):
    assert capi.load_library().dllm_cuda_beam_select(C.byref(_beam(**kw)), None) == rc


def test_beam_select_needs_a_descriptor():
    lib = capi.load_library()
    assert lib.dllm_cuda_beam_select(None, None) == INVALID
    assert lib.dllm_cuda_beam_workspace_bytes(None) == 0
    assert lib.dllm_cuda_beam_workspace_bytes(C.byref(_beam(batch=0))) == 0
    assert lib.dllm_cuda_beam_workspace_bytes(C.byref(_beam())) > 0


def _reorder(ptrs=(3 * P,), **kw):
    a = dict(batch=2, beams=4, parent=P, n=len(ptrs), tensors=(C.c_void_p * max(len(ptrs), 1))(*ptrs), row_stride=64,
             segs=1, seg_stride=0, run=64)
    a.update(kw)
    return capi.load_library().dllm_cuda_beam_reorder(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(batch=0), OK), (dict(ptrs=()), OK), (dict(segs=0), OK), (dict(run=0), OK),
    (dict(batch=-1), INVALID), (dict(beams=0), INVALID), (dict(n=-1), INVALID), (dict(segs=-1), INVALID),
    (dict(run=-1), INVALID), (dict(beams=129), UNSUPPORTED), (dict(parent=None), INVALID), (dict(tensors=None), INVALID),
    (dict(ptrs=(3 * P, None)), INVALID), (dict(ptrs=(3 * P, 2 * P, 3 * P)), INVALID),           # twice the same state
    (dict(ptrs=(2 * P,), parent=2 * P), INVALID),
    (dict(row_stride=63), INVALID), (dict(row_stride=0), INVALID), (dict(row_stride=-64), INVALID),
    (dict(segs=3, seg_stride=63), INVALID), (dict(segs=3, seg_stride=64, row_stride=128), INVALID),  # runs overlap
    (dict(segs=3, seg_stride=0, row_stride=192), INVALID),                            # a broadcast state
    (dict(segs=3, seg_stride=500, row_stride=64), INVALID),
])
def test_beam_reorder_refusals(kw, rc):
    assert _reorder(**kw) == rc


def test_struct_layout():
    assert C.sizeof(capi.BeamDesc) == 160
