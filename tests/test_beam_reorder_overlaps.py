"""States that share a byte are refused by dllm_cuda_beam_reorder and capi.beam_reorder, whatever their
layout; states that lie in one another's gaps are not."""
import ctypes as C

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from test_int8_beam_args import INVALID, P, _reorder

BASE = 1 << 20


def run_starts(base, rows, rs, segs, ss):
    return base + np.add.outer(np.arange(rows) * rs, np.arange(segs) * ss).ravel()


def share(a, b, la, lb):
    """whether a byte belongs to both states, by listing their bytes"""
    (rs, segs, ss, run), (rs2, segs2, ss2, run2) = la, lb
    x = (run_starts(a, 6, rs, segs, ss)[:, None] + np.arange(run)).ravel()
    y = (run_starts(b, 6, rs2, segs2, ss2)[:, None] + np.arange(run2)).ravel()
    return bool(np.intersect1d(x, y).size)


def layouts(rng):
    """a layout whose own runs do not overlap: rows around segments, or segments around rows"""
    run, segs = int(rng.integers(1, 9)), int(rng.integers(1, 5))
    inner = run + int(rng.integers(0, 12))
    if rng.random() < 0.5:
        return (segs - 1) * inner + run + int(rng.integers(0, 30)), segs, inner, run
    return inner, segs, 5 * inner + run + int(rng.integers(0, 30)), run


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused are launched: placeholders")
def test_states_of_one_call():
    """two states of one layout: refused where they share a byte, and only there (an accepted call fails at its
    launch, for there is no GPU)"""
    rng = np.random.default_rng(1)
    seen = [0, 0]
    for _ in range(6000):
        rs, segs, ss, run = la = layouts(rng)
        off = int(rng.integers(1, 8 * max(rs, ss) if segs > 1 else 8 * rs))
        ptrs = (BASE, BASE + off) if rng.random() < 0.5 else (BASE + off, BASE)
        rc = _reorder(ptrs=ptrs, batch=2, beams=3, row_stride=rs, segs=segs, seg_stride=ss, run=run)
        want = share(*ptrs, la, la)
        assert (rc == INVALID) == want, (la, off, rc, want)
        seen[want] += 1
    assert min(seen) > 500, seen


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused are launched: placeholders")
def test_parents_inside_a_state():
    rng = np.random.default_rng(2)
    seen = [0, 0]
    for _ in range(1500):
        rs, segs, ss, run = layouts(rng)
        at = BASE + int(rng.integers(-30, 6 * rs))
        bytes_of = (run_starts(BASE, 6, rs, segs, ss)[:, None] + np.arange(run)).ravel()
        want = bool(((bytes_of >= at) & (bytes_of < at + 24)).any())
        rc = _reorder(ptrs=(BASE,), parent=at, batch=2, beams=3, row_stride=rs, segs=segs, seg_stride=ss, run=run)
        assert (rc == INVALID) == want, (rs, segs, ss, run, at - BASE)
        seen[want] += 1
    assert min(seen) > 100, seen


def test_many_states_are_compared_quickly():
    """no state of many layers costs more than comparing its address"""
    ptrs = tuple(BASE + 4096 * i for i in range(200)) + (BASE + 4096 * 100 + 64,)
    assert _reorder(ptrs=ptrs, parent=P, row_stride=128, run=128) == INVALID


def test_states_of_two_layouts():
    rng = np.random.default_rng(3)
    seen = [0, 0]
    for _ in range(3000):
        la, lb = layouts(rng), layouts(rng)
        if la == lb:
            continue
        off = int(rng.integers(-200, 400))
        want = share(BASE, BASE + off, la, lb)
        groups = {la: [BASE], lb: [BASE + off, BASE + 100000]}
        if want:
            with pytest.raises(capi.DllmError, match="overlap"):
                capi._refuse_overlaps(groups, 6)
        else:
            capi._refuse_overlaps(groups, 6)
        seen[want] += 1
    assert min(seen) > 300, seen


@pytest.mark.gpu
def test_views_of_one_buffer():
    dev = torch.device("cuda", 0)
    p = torch.tensor([[1, 1, 3, 0], [2, 2, 2, 2]], dtype=torch.int32, device=dev)
    t = torch.arange(8 * 3 * 20, dtype=torch.float32, device=dev).view(8, 3, 20)
    start = t.clone()
    for states in ([t[:, :, :8], t[:, :, 4:12]],        # one layout
                   [t[:, :, :8], t[:, :, 4:]],          # two
                   [t, t[:, 1:2]],
                   [t[:, :2], t[:, 1:]],
                   [t[:, 1, :5], t[:, :, 4:6]]):
        with pytest.raises(capi.DllmError):
            capi.beam_reorder(states, p)
    assert torch.equal(t, start)
    inside = torch.zeros(8, 3, dtype=torch.int32, device=dev)
    with pytest.raises(capi.DllmError):
        capi.beam_reorder([inside], inside.view(-1)[8:16].view(2, 4))
    # in one another's gaps: each is moved
    src = [1, 1, 3, 0, 6, 6, 6, 6]
    for states in ([t[:, :, :8], t[:, :, 8:16]], [t[:, 0, :7], t[:, 1:, 3:9], t[:, 0, 7:]],
                   [t[:, :, i::4] for i in range(4)], [t[:, 0], t[:, 1], t[:, 2]]):
        t.copy_(start)
        want = [s[src] for s in states]
        capi.beam_reorder(states, p)
        assert all(torch.equal(s, w) for s, w in zip(states, want))
