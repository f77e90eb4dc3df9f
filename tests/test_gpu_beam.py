"""One step of beam search on the GPU (dllm_cuda_beam_select, dllm_cuda_beam_reorder) against its
definition in 64 bits.

Tolerance of a score.  The row's exponential sum is formed in fp32 pieces: each term has the
exponential's relative error (2^-22) and that of its argument (a rounding or three of 2^-24 on
|x - max|, whose mean under the softmax is at most log(vocab) < 13; the constant's own rounding adds
2^-26 of that), pieces of 32 terms are added in fp32 (31 x 2^-24), and a rescale or two add 2^-22 each:
below 4 + 39 + 4 + 31 + 8 < 96 x 2^-24 on the logarithm.  The score is rounded once (2^-24 of it).
Choices are exact where the ranks of the definition are further apart than twice that; within a
beam they are always exact."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from util import pack_mask

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
TOL = 96 * 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, scores, k, allow=None, finished=None, eos=-1, lengths=None, alpha=0.0):
    """(score, rank, parent, token) of the k best in the operator's order, and each beam's status."""
    x = x.detach().cpu().double().numpy()
    scores = scores.cpu().double().numpy()
    B, K = scores.shape
    V = x.shape[1]
    x = x.reshape(B, K, V).copy()
    if allow is not None:
        x[~allow.reshape(B, K, V)] = -np.inf
    out, status = [], np.zeros((B, K), np.int32)
    for s in range(B):
        cands = []  # (-rank, beam, -logit, id, score)
        for b in range(K):
            sc = scores[s, b]
            done = finished is not None and bool(finished[s, b])
            n = max((int(lengths[s, b]) if lengths is not None else 0) + (0 if done else 1), 1)
            div = float(n) ** alpha if alpha != 0 else 1.0
            if np.isnan(sc) or sc == np.inf:
                status[s, b] = capi.ROW_ERR_NONFINITE
                continue
            if sc == -np.inf:
                continue
            if done:
                cands.append((-sc / div, b, 0.0, eos, sc))
                continue
            row = x[s, b]
            if np.isnan(row).any() or (row == np.inf).any():
                status[s, b] = capi.ROW_ERR_NONFINITE
                continue
            m = row.max()
            if m == -np.inf:
                continue
            lse = m + np.log(np.exp(row - m).sum())
            order = np.lexsort((np.arange(V), -row))[:k]
            cands += [(-(sc + (row[i] - lse)) / div, b, -row[i], int(i), sc + (row[i] - lse)) for i in order
                      if row[i] > -np.inf]
        cands.sort()
        out.append([(c[4], -c[0], c[1], c[3]) for c in cands])
    return out, status


def check(got, ref, k, exact=False):
    score, parent, token = (t.cpu().numpy() for t in got)
    assert score.shape == parent.shape == token.shape == (len(ref), k)
    for s, cands in enumerate(ref):
        n = min(k, len(cands))
        assert (score[s, n:] == -np.inf).all() and (parent[s, n:] == -1).all() and (token[s, n:] == -1).all()
        pairs = [(int(p), int(t)) for p, t in zip(parent[s, :n], token[s, :n])]
        want = [(c[2], c[3]) for c in cands[:n]]
        if pairs != want:
            assert not exact, (s, pairs, want)
            at = {(c[2], c[3]): c for c in cands}
            assert len(set(pairs)) == n
            for i, p in enumerate(pairs):  # only neighbours closer than the tolerance may change places
                if p != want[i]:
                    assert p in at and abs(at[p][1] - cands[i][1]) <= 2 * TOL, (s, i, p, want[i])
        at = {(c[2], c[3]): c[0] for c in cands}
        want_score = np.array([at[p] for p in pairs])
        bad = np.abs(score[s, :n] - want_score) > TOL + 2.0 ** -24 * np.abs(want_score)
        assert not bad.any(), (s, score[s, :n][bad], want_score[bad])


def rows(rng, n, V, dtype, sd=2.0):
    x = rng.standard_normal((n, V)) * sd
    x[:, rng.integers(0, V, 8)] += 6
    return torch.from_numpy(x.astype(np.float32)).to(dtype).to(DEV)


def beam_scores(rng, B, K):
    return torch.from_numpy(-np.cumsum(rng.random((B, K)) * 3, 1).astype(np.float32)).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,k", [
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 4), (1, 4, 100, 8), (3, 2, 1000, 2), (1, 4, 32000, 8), (2, 5, 8191, 10),
    (1, 4, 128256, 8), (5, 8, 50257, 16), (40, 4, 4099, 4), (2, 16, 20000, 32), (1, 64, 3000, 128), (1, 128, 2000, 256),
    (1, 2, 151936, 256), (300, 1, 2049, 1), (1, 1, 262144, 1),
])
def test_select(dtype, B, K, V, k):
    rng = np.random.default_rng(B * 1000 + K * 100 + V)
    x, sc = rows(rng, B * K, V, dtype), beam_scores(rng, B, K)
    st = torch.full((B, K), 9, dtype=torch.int32, device=DEV)
    got = capi.beam_select(x, sc, k, status=st)
    ref, status = reference(x, sc, k)
    check(got, ref, k)
    np.testing.assert_array_equal(st.cpu().numpy(), status)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("frac", [0.5, 0.02, 0.0005])
@pytest.mark.parametrize("V", [33, 5000, 40003])
def test_select_masked(dtype, frac, V):
    rng = np.random.default_rng(V)
    B, K, k = 3, 4, 8
    x, sc = rows(rng, B * K, V, dtype), beam_scores(rng, B, K)
    allow = rng.random((B * K, V)) < frac
    allow[1] = False                # a row with nothing allowed
    allow[4:8] = False              # a sequence with nothing allowed
    allow[9] = False
    allow[9, V - 1] = True          # one id
    # what the mask leaves out may be anything
    hidden = torch.from_numpy(~allow).to(DEV)
    for junk in (float("nan"), float("inf"), -float("inf"), float(torch.finfo(dtype).min)):
        pick = torch.from_numpy(rng.random((B * K, V)) < 0.2).to(DEV)
        x = torch.where(hidden & pick, torch.full_like(x, junk), x)
    mask = torch.from_numpy(pack_mask(allow).view(np.int32)).to(DEV)
    st = torch.zeros(B, K, dtype=torch.int32, device=DEV)
    got = capi.beam_select(x, sc, k, mask=mask, status=st)
    check(got, reference(x, sc, k, allow)[0], k)
    assert (st == 0).all()


@pytest.mark.parametrize("alpha", [0.0, 0.6, 1.0, 2.0, -0.5])
def test_select_ended_beams_and_lengths(alpha):
    rng = np.random.default_rng(17)
    B, K, V = 6, 5, 3001
    x, sc = rows(rng, B * K, V, torch.float32), beam_scores(rng, B, K)
    fin = torch.from_numpy((rng.random((B, K)) < 0.4)).to(DEV)
    fin[2] = True                   # every beam ended
    x[fin.view(-1)] = float("nan")  # the logits of ended beams are not read
    ln = torch.from_numpy(rng.integers(0, 30, (B, K)).astype(np.int32)).to(DEV)
    sc[3, 1:] = -float("inf")
    of, ol = torch.empty(B, K, dtype=torch.uint8, device=DEV), torch.empty(B, K, dtype=torch.int32, device=DEV)
    got = capi.beam_select(x, sc, K, finished=fin, eos=7, lengths=ln, length_penalty=alpha, out_finished=of,
                           out_lengths=ol)
    ref, _ = reference(x, sc, K, None, fin.cpu().numpy(), 7, ln.cpu().numpy(), alpha)
    check(got, ref, K)
    parent, token = got[1].cpu().long(), got[2].cpu()
    p = parent.clamp(min=0)
    was = torch.gather(fin.cpu(), 1, p)
    assert torch.equal(of.cpu().bool(), (parent >= 0) & (was | (token == 7)))
    assert torch.equal(ol.cpu(), torch.where(parent >= 0, torch.gather(ln.cpu(), 1, p) + (~was).int(), torch.zeros_like(p).int()))


@pytest.mark.parametrize("dtype", TYPES)
def test_select_ties_go_to_the_lowest_index(dtype):
    B, K, V, k = 1, 3, 30000, 16
    x = torch.zeros(B * K, V, dtype=dtype, device=DEV)
    sc = torch.zeros(B, K, device=DEV)
    got = capi.beam_select(x, sc, k)                       # everything equal
    assert got[1].tolist() == [[0] * 16] and got[2].tolist() == [list(range(16))]
    x[:, 1::2] = -0.0                                      # the two zeros are the same value
    got = capi.beam_select(x, sc, k)
    assert got[1].tolist() == [[0] * 16] and got[2].tolist() == [list(range(16))]
    x.zero_()
    x[:, 29990:] = 1.0                                     # ten of each beam, at the end
    got = capi.beam_select(x, sc, k)
    assert got[1].tolist() == [[0] * 10 + [1] * 6]
    assert got[2].tolist() == [list(range(29990, 30000)) + list(range(29990, 29996))]
    rng = np.random.default_rng(8)
    x = torch.from_numpy(rng.integers(-3, 4, (B * K, V)).astype(np.float32)).to(dtype).to(DEV)  # many equal logits
    sc = torch.tensor([[-1.0, -1.0, -1.5]], device=DEV)
    check(capi.beam_select(x, sc, 256), reference(x, sc, 256)[0], 256, exact=True)


@pytest.mark.parametrize("kind", ["rising", "falling", "blocks", "few", "denormal", "wide"])
@pytest.mark.parametrize("k", [1, 8, 100])
def test_select_orders_of_values(kind, k):
    """rows in which a running threshold fails: every entry is a candidate, or almost none"""
    rng = np.random.default_rng(21)
    V, K = 70000, 2
    v = np.sort(rng.standard_normal((K, V)) * 3, axis=1)
    if kind == "falling":
        v = v[:, ::-1]
    elif kind == "blocks":
        v = np.repeat(np.arange(V // 1000) * 0.1, 1000)[None, :] + np.zeros((K, 1))
    elif kind == "few":
        v = np.full((K, V), -np.inf)
        v[:, rng.integers(0, V, 5)] = rng.standard_normal(5)
    elif kind == "denormal":
        v = rng.integers(-50, 50, (K, V)) * 1e-45
    elif kind == "wide":
        v = rng.standard_normal((K, V)) * 1e30
        v[:, ::7] = np.finfo(np.float32).min
    x = torch.from_numpy(np.ascontiguousarray(v).astype(np.float32)).to(DEV)
    sc = torch.tensor([[-0.5, -0.75]], device=DEV)
    check(capi.beam_select(x, sc, k), reference(x, sc, k)[0], k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", ["lowest", "highest", -1e6, 2.0 ** 20, 3e4])
def test_select_log_probabilities_of_huge_logits(dtype, value):
    """equal logits have the probability 1 / n, however large they are"""
    V = 5000
    v = {"lowest": torch.finfo(dtype).min, "highest": torch.finfo(dtype).max}.get(value, value)
    if abs(v) > torch.finfo(dtype).max:
        pytest.skip("not a number of this type")
    x = torch.full((2, V), v, dtype=dtype, device=DEV)
    allow = np.zeros((2, V), bool)
    allow[:, 7:4000:31] = True
    mask = torch.from_numpy(pack_mask(allow).view(np.int32)).to(DEV)
    for kw, n, ids in ((dict(), V, [0, 1, 2]), (dict(mask=mask), int(allow[0].sum()), [7, 38, 69])):
        got = capi.beam_select(x, torch.tensor([[-1.0, -1.5]], device=DEV), 3, **kw)
        assert got[1].tolist() == [[0, 0, 0]] and got[2].tolist() == [ids]
        assert (got[0].double().cpu() + 1 + np.log(n)).abs().max() <= TOL + 2.0 ** -24 * 11


@pytest.mark.parametrize("alpha", [1000.0, -1000.0, 40.0])
def test_select_extreme_length_penalty(alpha):
    """ranks stay finite: the choice is defined, and every slot is filled once"""
    rng = np.random.default_rng(3)
    x, sc = rows(rng, 8, 4000, torch.float32), beam_scores(rng, 2, 4)
    sc[0, 0] = 0.0
    ln = torch.tensor([[1, 50, 100000, 7], [0, 0, 3, 3]], dtype=torch.int32, device=DEV)
    score, parent, token = capi.beam_select(x, sc, 6, lengths=ln, length_penalty=alpha)
    assert (parent >= 0).all() and torch.isfinite(score).all()
    for s in range(2):
        assert len({(int(p), int(t)) for p, t in zip(parent[s], token[s])}) == 6


def test_select_nonfinite_rows_and_scores():
    rng = np.random.default_rng(5)
    x, sc = rows(rng, 8, 9000, torch.float32), beam_scores(rng, 2, 4)
    x[0, 8999] = float("nan")
    x[2, 0] = float("inf")
    x[3, 100:200] = -float("inf")
    x[5] = -float("inf")
    x[6] = float("nan")
    sc[1, 0], sc[1, 3] = float("nan"), float("inf")
    st = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    got = capi.beam_select(x, sc, 8, status=st)
    ref, status = reference(x, sc, 8)
    check(got, ref, 8)
    np.testing.assert_array_equal(st.cpu().numpy(), status)
    assert st.tolist() == [[2, 0, 2, 0], [2, 0, 2, 2]] and (got[1][1] == -1).all()


def test_select_first_step_and_dead_sequences():
    rng = np.random.default_rng(6)
    x, sc = rows(rng, 12, 3000, torch.bfloat16), torch.zeros(3, 4, device=DEV)
    sc[:, 1:] = -float("inf")
    sc[1] = -float("inf")
    got = capi.beam_select(x, sc, 8)
    check(got, reference(x, sc, 8)[0], 8)
    assert (got[1][0] == 0).all() and (got[1][1] == -1).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,base,stride", [(1000, 1, 1001), (4097, 3, 4100), (777, 5, 1024), (16, 7, 17), (40000, 2, 40009)])
def test_select_strides(dtype, V, base, stride):
    rng = np.random.default_rng(V)
    n = 6
    buf = torch.full((base + n * stride + 64,), 50.0, dtype=dtype, device=DEV)  # what lies around would win
    x = buf[base:].as_strided((n, V), (stride, 1))
    x.copy_(rows(rng, n, V, dtype))
    allow = rng.random((n, V)) < 0.5
    W = (V + 31) // 32
    wide = torch.full((n, W + 3), -1, dtype=torch.int32, device=DEV)
    wide[:, :W] = torch.from_numpy(pack_mask(allow).view(np.int32)).to(DEV)
    sc = beam_scores(rng, 2, 3)
    check(capi.beam_select(x, sc, 6), reference(x, sc, 6)[0], 6)
    check(capi.beam_select(x, sc, 6, mask=wide), reference(x, sc, 6, allow)[0], 6)


def test_select_outputs_over_inputs():
    rng = np.random.default_rng(9)
    B, K, V = 7, 6, 5000
    x, sc = rows(rng, B * K, V, torch.float32), beam_scores(rng, B, K)
    fin = torch.from_numpy((rng.random((B, K)) < 0.3).astype(np.uint8)).to(DEV)
    ln = torch.from_numpy(rng.integers(1, 9, (B, K)).astype(np.int32)).to(DEV)
    of, ol = torch.empty_like(fin), torch.empty_like(ln)
    kw = dict(eos=3, length_penalty=0.7)
    want = capi.beam_select(x, sc, K, finished=fin, lengths=ln, out_finished=of, out_lengths=ol, **kw)
    s2, f2, l2 = sc.clone(), fin.clone(), ln.clone()
    p, t = torch.empty(B, K, dtype=torch.int32, device=DEV), torch.empty(B, K, dtype=torch.int32, device=DEV)
    capi.beam_select(x, s2, K, finished=f2, lengths=l2, out=(s2, p, t), out_finished=f2, out_lengths=l2, **kw)
    for a, b in zip((*want, of, ol), (s2, p, t, f2, l2)):
        assert torch.equal(a, b)


def test_select_empty_batch():
    got = capi.beam_select(torch.empty(0, 100, device=DEV), torch.empty(0, 4, device=DEV), 8)
    assert [t.shape for t in got] == [(0, 8)] * 3


def test_select_far_rows():
    """a row whose offset passes 2^31 elements"""
    V, stride = 1000, 2 ** 30 + 7
    buf = torch.empty(3 * stride + V, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((4, V), (stride, 1))
    rng = np.random.default_rng(2)
    x.copy_(rows(rng, 4, V, torch.bfloat16))
    sc = beam_scores(rng, 1, 4)
    check(capi.beam_select(x, sc, 8), reference(x, sc, 8)[0], 8)


def test_select_graph_and_streams():
    rng = np.random.default_rng(10)
    xs = [rows(rng, 8, 20000, torch.float32) for _ in range(3)]
    sc = beam_scores(rng, 2, 4)
    want = [[t.clone() for t in capi.beam_select(x, sc, 8)] for x in xs]
    x = xs[0].clone()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    out = tuple(torch.empty(2, 8, dtype=d, device=DEV) for d in (torch.float32, torch.int32, torch.int32))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.beam_select(x, sc, 8, out=out, workspace=ws)
    for i in (1, 2, 0):
        x.copy_(xs[i])
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, capi.beam_select(xs[i], sc, 8)))
    torch.cuda.synchronize()
    for i, o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want[i]))


def test_select_capture_without_a_workspace_is_refused():
    import ctypes as C

    x, sc = torch.zeros(4, 100, device=DEV), torch.zeros(1, 4, device=DEV)
    d, out = capi.fill_beam_desc(x, sc, 4)
    assert not d.workspace
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        x.add_(1)
        rc = capi.load_library().dllm_cuda_beam_select(C.byref(d), torch.cuda.current_stream().cuda_stream)
    assert rc == capi.DLLM_ERR_INVALID_ARG
    g.replay()
    assert capi.load_library().dllm_cuda_beam_select(C.byref(d), torch.cuda.current_stream().cuda_stream) == capi.DLLM_OK
    torch.cuda.synchronize()
    assert out[2].tolist() == [[0, 1, 2, 3]]


def test_select_tensor_refusals():
    x, sc = torch.zeros(8, 100, device=DEV), torch.zeros(2, 4, device=DEV)
    for call in (
        lambda: capi.beam_select(x[:7], sc, 4),
        lambda: capi.beam_select(x.double(), sc, 4),
        lambda: capi.beam_select(x.cpu(), sc, 4),
        lambda: capi.beam_select(x, sc.cpu(), 4),
        lambda: capi.beam_select(x, sc.double(), 4),
        lambda: capi.beam_select(x.t(), torch.zeros(25, 4, device=DEV), 4),
        lambda: capi.beam_select(x, sc, 0),
        lambda: capi.beam_select(x, sc, 257),
        lambda: capi.beam_select(x, sc, 4, mask=torch.zeros(8, 3, dtype=torch.int32, device=DEV)),
        lambda: capi.beam_select(x, sc, 4, finished=torch.zeros(2, 4, dtype=torch.int32, device=DEV), eos=1),
        lambda: capi.beam_select(x, sc, 4, finished=torch.zeros(2, 4, dtype=torch.uint8, device=DEV)),
        lambda: capi.beam_select(x, sc, 4, length_penalty=1.0),
        lambda: capi.beam_select(x, sc, 4, out=(sc, sc, sc)),
        lambda: capi.beam_select(x, sc, 4, workspace=torch.empty(16, dtype=torch.uint8, device=DEV)),
    ):
        with pytest.raises(capi.DllmError):
            call()


# ---- states after their parents --------------------------------------------------------------

def moved(t, parents):
    B, K = parents.shape
    p = parents.cpu().long()
    ok = (p >= 0) & (p < K)
    src = torch.arange(B)[:, None] * K + torch.where(ok, p, torch.arange(K).expand(B, K))
    return t.index_select(0, src.reshape(-1).to(t.device))


def parents_of(rng, B, K, kind):
    j = np.arange(K)
    p = {"random": rng.integers(0, K, (B, K)), "same": np.tile(j, (B, 1)), "one": np.zeros((B, K)),
         "cycle": np.tile((j + 1) % K, (B, 1)), "reverse": np.tile(j[::-1], (B, 1)),
         "holes": np.where(rng.random((B, K)) < 0.4, -1, rng.integers(0, K, (B, K))),
         "out of range": np.where(rng.random((B, K)) < 0.4, rng.integers(K, 2 ** 31 - 1, (B, K)), rng.integers(0, K, (B, K)))}[kind]
    return torch.from_numpy(p.astype(np.int32)).to(DEV)


@pytest.mark.parametrize("kind", ["random", "same", "one", "cycle", "reverse", "holes", "out of range"])
@pytest.mark.parametrize("B,K", [(1, 1), (1, 2), (3, 4), (2, 9), (1, 33), (2, 128)])
def test_reorder(kind, B, K):
    rng = np.random.default_rng(K)
    p = parents_of(rng, B, K, kind)
    for dtype, shape in ((torch.float32, (100,)), (torch.bfloat16, (3, 64)), (torch.int32, (511,)), (torch.uint8, (37,)),
                         (torch.int64, ()), (torch.float16, (5000,))):
        t = torch.randint(0, 100, (B * K, *shape), device=DEV).to(dtype)
        want = moved(t, p)
        capi.beam_reorder([t], p)
        assert torch.equal(t, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
@pytest.mark.parametrize("length", [1, 7, 100, 256])
@pytest.mark.parametrize("dim", [1, 40, 64])
def test_reorder_cache_views(dtype, length, dim):
    """the used part of caches [rows][heads][capacity][dim]; the rest stays as it was"""
    rng = np.random.default_rng(length)
    B, K, H, cap = 2, 5, 3, 256
    p = parents_of(rng, B, K, "random")
    full = [torch.randint(0, 100, (B * K, H, cap, dim), device=DEV).to(dtype) for _ in range(5)]
    want = [t.clone() for t in full]
    for t in want:
        t[:, :, :length] = moved(t[:, :, :length], p)
    capi.beam_reorder([t[:, :, :length] for t in full], p)
    assert all(torch.equal(a, b) for a, b in zip(full, want))


@pytest.mark.parametrize("dtype,length", [(torch.bfloat16, 101), (torch.bfloat16, 7), (torch.float32, 99), (torch.uint8, 1),
                                          (torch.uint8, 4099)])
def test_reorder_short_last_vector(dtype, length):
    """runs that start on multiples of 16 bytes and end between them: what follows a run stays as it was"""
    rng = np.random.default_rng(length)
    p = parents_of(rng, 3, 6, "random")
    full = torch.randint(0, 100, (18, 2, 8192), device=DEV).to(dtype)
    want = full.clone()
    want[:, :, :length] = moved(full[:, :, :length], p)
    capi.beam_reorder([full[:, :, :length]], p)
    assert torch.equal(full, want)


def test_reorder_other_layouts():
    rng = np.random.default_rng(1)
    B, K = 3, 4
    p = parents_of(rng, B, K, "random")
    both = torch.randn(B * K, 2, 6, 50, device=DEV)                 # keys and values of one buffer
    layers = torch.randn(5, B * K, 33, device=DEV)                  # rows inside layers
    odd = torch.randn(B * K * 61 + 3, device=DEV)[3:].view(B * K, 61)
    wide = torch.randn(B * K, 64, device=DEV)[:, ::2]               # runs of one element
    empty = torch.empty(B * K, 0, device=DEV)
    states = [both[:, 0], both[:, 1], layers.transpose(0, 1), odd, wide, empty, torch.randn(B * K, 1, 1, device=DEV)]
    want = [moved(t, p) for t in states]
    capi.beam_reorder(states, p)
    for a, b in zip(states, want):
        assert torch.equal(a, b)
    capi.beam_reorder([], p)


def test_reorder_many_tensors_and_large_rows():
    rng = np.random.default_rng(4)
    p = parents_of(rng, 2, 3, "random")
    ts = [torch.randn(6, 40, device=DEV) for _ in range(150)]
    want = [moved(t, p) for t in ts]
    capi.beam_reorder(ts, p)
    assert all(torch.equal(a, b) for a, b in zip(ts, want))
    t = torch.empty(6, 2 ** 29 + 16, dtype=torch.uint8, device=DEV)  # offsets pass 2^31 bytes
    for i in range(6):
        t[i].fill_(i)
        t[i, -5:] = 50 + i
    capi.beam_reorder([t], p)
    src = moved(torch.arange(6, device=DEV), p).tolist()
    for i in range(6):
        assert (t[i, :-5] == src[i]).all() and (t[i, -5:] == 50 + src[i]).all()


def test_reorder_graph():
    rng = np.random.default_rng(3)
    p = parents_of(rng, 2, 4, "random")
    t = torch.randn(8, 1000, device=DEV)
    start = t.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.beam_reorder([t], p)
    for kind in ("cycle", "random"):
        t.copy_(start)
        p.copy_(parents_of(rng, 2, 4, kind))
        g.replay()
        g.replay()
        assert torch.equal(t, moved(moved(start, p), p))


def test_reorder_refusals():
    p = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    t = torch.zeros(8, 30, device=DEV)
    for call in (
        lambda: capi.beam_reorder([t[:7]], p),
        lambda: capi.beam_reorder([t.cpu()], p),
        lambda: capi.beam_reorder([t], p.long()),
        lambda: capi.beam_reorder([t], p.cpu()),
        lambda: capi.beam_reorder([t], p.t()),
        lambda: capi.beam_reorder([t, t], p),
        lambda: capi.beam_reorder([p.view(8, 1)], p),
        lambda: capi.beam_reorder([t, t[:, :10]], p),
        lambda: capi.beam_reorder([torch.zeros(1, 30, device=DEV).expand(8, 30)], p),
        lambda: capi.beam_reorder([torch.zeros(8, 1, device=DEV).expand(8, 30)], p),
        lambda: capi.beam_reorder([torch.zeros(8, 4, 6, 10, device=DEV)[:, :, :5, :7]], p),
    ):
        with pytest.raises(capi.DllmError):
            call()
    assert (t == 0).all()


# ---- how the calls share memory --------------------------------------------------------------

def test_captured_calls_keep_their_scratch():
    """graphs captured without a workspace have scratch of their own: larger eager calls in between, which
    grow the eager scratch, and two graphs replayed at once on two streams do not disturb them"""
    rng = np.random.default_rng(31)
    xs = [rows(rng, 8, 30000, torch.float32) for _ in range(2)]
    sc = beam_scores(rng, 2, 4)
    want = [[t.clone() for t in capi.beam_select(x, sc, 8)] for x in xs]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(capi.beam_select(x, sc, 8))
        graphs.append(g)
    big = rows(rng, 64, 50000, torch.float32)
    capi.beam_select(big, beam_scores(rng, 8, 8), 64)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_stream_argument():
    rng = np.random.default_rng(32)
    x, sc = rows(rng, 8, 30000, torch.float32), beam_scores(rng, 2, 4)
    want = capi.beam_select(x, sc, 4)
    t = torch.randn(8, 100, device=DEV)
    after = moved(t, want[1])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = capi.beam_select(x, sc, 4, stream=s.cuda_stream)
    capi.beam_reorder([t], got[1], stream=s.cuda_stream)
    q, scale = capi.quantize_rows_i8(t, stream=s.cuda_stream)
    m = capi.matmul_i8(q, scale, q, scale, stream=s.cuda_stream)
    lg = capi.lmhead_logits_i8(t, q, scale, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(t, after)
    q2, scale2 = capi.quantize_rows_i8(t)
    assert torch.equal(q, q2) and torch.equal(m, capi.matmul_i8(q2, scale2, q2, scale2))
    assert torch.equal(lg, capi.lmhead_logits_i8(t, q2, scale2))
    assert torch.equal(capi.beam_select(x, sc, 4, stream=0)[2], want[2])
    assert torch.equal(capi.beam_select(logits=x, scores=sc, k=4, stream=s.cuda_stream)[2], want[2])


def test_calls_from_several_threads():
    import threading

    rng = np.random.default_rng(33)
    cases = [(rows(rng, 4 * n, 9000 * n, torch.float32), beam_scores(rng, n, 4)) for n in (1, 2, 3, 5)]
    want = [capi.beam_select(x, sc, 6) for x, sc in cases]
    bad = []

    def go(i):
        for _ in range(30):
            got = capi.beam_select(*cases[i], 6)
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)

    threads = [threading.Thread(target=go, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_subnormal_scores():
    """scores below the smallest normal number count, and an ended beam's is copied as it is"""
    sc = torch.from_numpy(np.ldexp(np.array([[-3.0, -2.0, -5.0, -1.0]]), -149).astype(np.float32)).to(DEV)
    x = torch.full((4, 100), float("-inf"), device=DEV)
    x[:, 9] = 4.0  # the only continuation, of log-probability 0
    done = torch.tensor([[0, 1, 1, 0]], dtype=torch.uint8, device=DEV)
    score, parent, token = capi.beam_select(x, sc, 4, finished=done, eos=3)
    assert parent.tolist() == [[3, 1, 0, 2]] and token.tolist() == [[9, 3, 9, 3]]
    np.testing.assert_array_equal(score.cpu().numpy(), sc.cpu().numpy()[:, [3, 1, 0, 2]])
