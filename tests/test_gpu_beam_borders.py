"""dllm_cuda_beam_select where its kernels change how they compute: logits around +-2^20, where the reference
of the exponential sums changes its form, and ranks that are equal only as exact quotients; and the order
within a beam, which is exact whatever the scores' tolerance.  Tolerance and reference are those of
test_gpu_beam."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from test_gpu_beam import DEV, TYPES, beam_scores, check, reference, rows
from util import pack_mask

pytestmark = pytest.mark.gpu

BORDER = 2.0 ** 20


def check_beams(got, ref):
    """the tokens of each beam are the first of its own candidates, in their order"""
    parent, token = (t.cpu().numpy() for t in got[1:])
    for s, cands in enumerate(ref):
        for b in set(parent[s].tolist()) - {-1}:
            mine = [c[3] for c in cands if c[2] == b]
            took = token[s][parent[s] == b].tolist()
            assert took == mine[:len(took)], (s, b, took, mine[:len(took)])


def crossing(rng, n, V, kind):
    """rows of logits on both sides of a border; neighbours are up to 1/8 apart, so that all count in the sum"""
    if kind == "up":          # most of the row below, the end above: a lane's maximum crosses late
        v = np.full((n, V), -BORDER - 0.125)
        v[:, V * 12 // 13:] = -BORDER + 0.0625
    elif kind == "scattered":  # a lane crosses at a tile of its own
        v = np.full((n, V), -BORDER - 0.25)
        v[rng.random((n, V)) < 0.002] = -BORDER + 0.1875
    elif kind == "steps":      # a lane's maximum rises tile by tile
        v = -BORDER - 1 + np.floor(np.arange(V) * 16 / V) / 8 + np.zeros((n, 1))
    elif kind == "around":
        v = -BORDER + rng.integers(-8, 9, (n, V)) / 8
    elif kind == "positive":
        v = BORDER - 1 + np.floor(np.arange(V) * 16 / V) / 8 + np.zeros((n, 1))
    elif kind == "both ends":  # -inf first, then from below the lower border
        v = np.full((n, V), -np.inf)
        v[:, V // 3:] = -BORDER - 0.125
        v[:, V * 2 // 3:] = -BORDER + 0.0625
    return v.astype(np.float32)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("kind", ["up", "scattered", "steps", "around", "positive", "both ends"])
def test_sums_across_the_border(kind, masked):
    """128 rows of 106496: a piece has five tiles or more"""
    rng = np.random.default_rng(20)
    B, K, V, k = 32, 4, 106496, 5
    x = torch.from_numpy(crossing(rng, B * K, V, kind)).to(DEV)
    sc = beam_scores(rng, B, K)
    allow, kw = None, {}
    if masked:
        allow = rng.random((B * K, V)) < 0.6
        kw["mask"] = torch.from_numpy(pack_mask(allow).view(np.int32)).to(DEV)
    got = capi.beam_select(x, sc, k, **kw)
    ref, _ = reference(x, sc, k, allow)
    check(got, ref, k)
    check_beams(got, ref)


@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_sums_across_the_border_in_bf16(sign):
    """neighbouring numbers are thousands apart there: only the largest count"""
    rng = np.random.default_rng(22)
    B, K, V, k = 32, 4, 200000, 5
    v = sign * BORDER * (1 + rng.integers(-6, 7, (B * K, V)) / 256)
    x = torch.from_numpy(v.astype(np.float32)).to(torch.bfloat16).to(DEV)
    sc = beam_scores(rng, B, K)
    got = capi.beam_select(x, sc, k)
    ref, _ = reference(x, sc, k)
    check(got, ref, k)
    check_beams(got, ref)


@pytest.mark.parametrize("ended", [True, False])
@pytest.mark.parametrize("beams", [2, 64, 128])
def test_ranks_are_quotients(beams, ended):
    """scores of -3 per token: with alpha = 1 every rank is -3 exactly, and the beams come in their order"""
    n = torch.arange(1, beams + 1, dtype=torch.int32, device=DEV).view(1, beams)
    x = torch.full((beams, 40), float("-inf"), device=DEV)
    x[:, 6] = 0.0  # the only continuation; its log-probability is exactly 0
    done = torch.full((1, beams), int(ended), dtype=torch.uint8, device=DEV)
    sc = -3.0 * n.float()
    score, parent, token = capi.beam_select(x, sc, beams, finished=done, eos=9, lengths=n if ended else n - 1,
                                            length_penalty=1.0)
    assert parent.tolist() == [list(range(beams))]
    assert torch.equal(score, sc) and (token == (9 if ended else 6)).all()


def test_a_score_below_the_range_of_fp32():
    """it is chosen, after the others, and its score is -inf"""
    x = torch.tensor([[3e38, -3e38, -float("inf")], [1.0, 1.0, 1.0]], device=DEV)
    sc = torch.tensor([[-2.0, -5.0]], device=DEV)
    score, parent, token = capi.beam_select(x, sc, 6)
    assert parent.tolist() == [[0, 1, 1, 1, 0, -1]] and token.tolist() == [[0, 0, 1, 2, 1, -1]]
    assert score[0, 0] == -2.0 and torch.isfinite(score[0, :4]).all() and (score[0, 4:] == -float("inf")).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,k,frac", [(2, 5, 8191, 10, 1.0), (1, 4, 128256, 8, 1.0), (5, 8, 50257, 16, 1.0),
                                          (1, 64, 3000, 128, 1.0), (1, 2, 151936, 256, 1.0), (3, 4, 40003, 8, 0.5),
                                          (40, 8, 30000, 16, 0.02)])
def test_the_order_within_a_beam_is_exact(dtype, B, K, V, k, frac):
    rng = np.random.default_rng(V)
    x, sc = rows(rng, B * K, V, dtype), beam_scores(rng, B, K)
    allow, kw = None, {}
    if frac < 1:
        allow = rng.random((B * K, V)) < frac
        kw["mask"] = torch.from_numpy(pack_mask(allow).view(np.int32)).to(DEV)
    got = capi.beam_select(x, sc, k, **kw)
    ref, _ = reference(x, sc, k, allow)
    check(got, ref, k)
    check_beams(got, ref)
