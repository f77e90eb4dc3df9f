"""What decode.BeamLoop says of a run that went wrong, eager and replayed, and its capture in a process in
which nothing has run before."""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from test_gpu_beam_loop import loop

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def results(bl):
    return [t.clone() for t in (bl.tokens, bl.scores, bl.lengths, bl.finished)]


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_hidden_states_that_are_not_finite(captured, value):
    bl, _ = loop(np.random.default_rng(1), 3, 4, 5, length_penalty=0.5)
    go = bl.replay if captured else bl.run_eager
    go()
    want = results(bl)
    assert torch.equal(bl.check(), want[0]) and (bl.status == 0).all()
    good = bl.ring[1, 4:8, 7].clone()
    bl.ring[1, 4:8, 7] = value  # every beam of the second sequence, in steps 1 and 4
    go()
    assert (bl.status[1] == capi.ROW_ERR_NONFINITE).all() and (bl.status[[0, 2]] == 0).all()
    with pytest.raises(capi.DllmError, match=r"\[1\]"):
        bl.check()
    for got, t in zip(results(bl), want):  # the other sequences are as before
        assert torch.equal(got[0], t[0]) and torch.equal(got[2], t[2])
    assert (bl.tokens[1, :, 1:] == -1).all() and (bl.scores[1] == -float("inf")).all()
    bl.ring[1, 4:8, 7] = good
    go()
    bl.check()
    assert all(torch.equal(a, b) for a, b in zip(results(bl), want))


def test_one_beam_that_is_not_finite():
    """it offers nothing and is named; the others of its sequence go on"""
    bl, _ = loop(np.random.default_rng(2), 2, 4, 3)
    bl.ring[2, 6, 0] = float("nan")  # in the last step, the third beam of the second sequence
    bl.run_eager()
    assert bl.status.tolist() == [[0] * 4, [0, 0, capi.ROW_ERR_NONFINITE, 0]]
    assert (bl.tokens >= 0).all() and torch.isfinite(bl.scores).all() and (bl.parents[1] != 2).all()
    with pytest.raises(capi.DllmError, match="not finite"):
        bl.check()


@pytest.mark.parametrize("captured", [False, True])
def test_a_wait_that_runs_out(captured):
    """the issuing threads of the LM head's product wait for something that nothing completes (the library's test
    hook): the run ends, and neither tokens nor scores look like results"""
    bl, _ = loop(np.random.default_rng(3), 2, 3, 4)
    want = bl.run_eager().clone()
    bl.check()
    capi.inject_wait_timeout(capi.FAULT_PRODUCT_WAIT, 1000)
    try:
        bl.capture().replay() if captured else bl.run_eager()
        torch.cuda.synchronize()
    finally:
        capi.inject_wait_timeout(capi.FAULT_NONE)
    assert (bl.status & capi.ROW_ERR_TIMEOUT).all()
    assert (bl.tokens == -1).all() and torch.isnan(bl.scores).all()
    with pytest.raises(capi.DllmError, match="ran out"):
        bl.check()
    bl.capture().replay() if captured else bl.run_eager()  # a graph keeps the hook that it was captured with
    assert torch.equal(bl.check(), want)


@pytest.mark.parametrize("masked", [False, True])
def test_capture_in_a_new_process(masked):
    """nothing has run before the capture: no kernel is loaded, no attribute set"""
    script = f"""
import sys
sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, 'tests')!r}, {os.path.join(ROOT, 'oracle')!r}]
import numpy as np, torch
from test_gpu_beam_loop import loop
bl, _ = loop(np.random.default_rng(4), 2, 4, 6, length_penalty=0.6, masked={masked})
start = [t.clone() for t in bl.states]
got = bl.capture().replay().clone()
bl.check()
after = [t.clone() for t in (bl.scores, bl.lengths, *bl.states)]
for t, s in zip(bl.states, start):
    t.copy_(s)
assert torch.equal(bl.run_eager(), got)
assert all(torch.equal(a, b) for a, b in zip((bl.scores, bl.lengths, *bl.states), after))
print("the same")
"""
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]
