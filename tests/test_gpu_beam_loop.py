"""decode.BeamLoop: LM head with int8 weights, selection, states moved after their parents, step after
step, against the definition of each step in 64 bits on the state that the loop holds; and its
capture as a CUDA graph."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from diskllm_b200.decode import BeamLoop
from test_gpu_beam import check, moved, reference
from test_gpu_int8 import check_product, ref_matmul, ref_quantize
from util import pack_mask

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def loop(rng, batch, beams, steps, hidden=128, vocab=900, masked=False, **kw):
    ring = torch.from_numpy(rng.standard_normal((3, batch * beams, hidden)).astype(np.float32)).to(DEV)
    wq, ws = capi.quantize_rows_i8(torch.from_numpy((0.3 * rng.standard_normal((vocab, hidden))).astype(np.float32)).to(DEV))
    states = [torch.randn(batch * beams, 2, 16, 8, device=DEV)[:, :, :11],
              torch.randint(0, 99, (batch * beams, 5), dtype=torch.int32, device=DEV)]
    allow = None
    if masked:
        allow = rng.random((3, batch * beams, vocab)) < 0.1
        kw["mask_ring"] = torch.stack([torch.from_numpy(pack_mask(a).view(np.int32)) for a in allow]).to(DEV)
    return BeamLoop(ring, wq, ws, batch, beams, steps, states=states, eos=5, **kw), allow


@pytest.mark.parametrize("batch,beams,masked,alpha", [(1, 1, False, 0.0), (2, 4, False, 0.7), (3, 5, True, 1.0)])
def test_every_step(batch, beams, masked, alpha):
    rng = np.random.default_rng(beams)
    nw = torch.from_numpy((1 + 0.1 * rng.standard_normal(128)).astype(np.float32)).to(DEV)
    bl, allow = loop(rng, batch, beams, 6, masked=masked, length_penalty=alpha, norm_w=nw, softcap=20.0)
    bl._reset()
    hist = torch.empty(batch * beams, 0, dtype=torch.int32, device=DEV)
    for i in range(6):
        if i == 2:  # a beam ends, so that the following steps hold one that has
            bl.finished[0, -1] = 1
        before = [t.clone() for t in (bl.scores, bl.finished, bl.lengths, *bl.states)]
        bl._step(i)
        q, s = ref_quantize(bl.ring[i % 3], True, nw)
        lg = ref_matmul(torch.from_numpy(q), torch.from_numpy(s), bl.wq, bl.w_scale, 20.0)
        check_product(bl.logits, lg, torch.float32)
        sc, fin, ln = before[:3]
        ref, _ = reference(bl.logits, sc, beams, None if allow is None else allow[i % 3], fin.cpu().numpy(), 5,
                           ln.cpu().numpy(), alpha)
        check((bl.scores, bl.parents, bl.new), ref, beams)
        for t, old in zip(bl.states, before[3:]):
            assert torch.equal(t, moved(old, bl.parents))
        hist = torch.cat([moved(hist, bl.parents), bl.new.view(-1, 1)], 1)
        assert torch.equal(bl.hist[:, :i + 1], hist)


@pytest.mark.parametrize("masked", [False, True])
def test_graph_replay_equals_eager(masked):
    bl, _ = loop(np.random.default_rng(4), 2, 4, 8, length_penalty=0.6, masked=masked)
    start = [t.clone() for t in bl.states]
    want = bl.run_eager().clone()
    results = [t.clone() for t in (bl.scores, bl.lengths, bl.finished, *bl.states)]
    for _ in range(2):
        for t, s in zip(bl.states, start):
            t.copy_(s)
        got = bl.replay() if bl.graph else bl.capture().replay()
        assert torch.equal(got, want)
        for a, b in zip((bl.scores, bl.lengths, bl.finished, *bl.states), results):
            assert torch.equal(a, b)


def test_scores_are_those_of_the_tokens():
    """a beam's score is the sum of the log-probabilities of its own tokens"""
    bl, _ = loop(np.random.default_rng(6), 1, 3, 4)
    bl.ring[:, 1:] = bl.ring[:, :1]  # hidden states that do not depend on the beam: any token path can be scored
    bl.run_eager()
    lp = []
    for i in range(4):
        lg = capi.lmhead_logits_i8(bl.ring[i % 3], bl.wq, bl.w_scale)[0].double()
        lp.append((lg - lg.logsumexp(0)).cpu())
    for b in range(3):
        toks = bl.tokens[0, b].tolist()
        n = toks.index(5) + 1 if 5 in toks else 4
        want = sum(float(lp[i][t]) for i, t in enumerate(toks[:n]))
        # each step's score is off by at most 96 x 2^-24 + 2^-24 of itself
        assert abs(float(bl.scores[0, b]) - want) <= 4 * (96 + abs(want)) * 2.0 ** -24
        assert toks[n:] == [5] * (4 - n) and int(bl.lengths[0, b]) == n
