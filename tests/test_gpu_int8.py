"""The int8 LM head on the GPU (dllm_cuda_quantize_rows_i8, dllm_cuda_matmul_i8,
dllm_cuda_lmhead_logits_i8) against their definitions in 64 bits.

Tolerances.  Codes and scales: none; both sides decide them in 64 bits, whose rounding (2^-53) moves
a quotient over a half-integer for about one in 10^13 values.  Products: the integer sum is exact;
its conversion to fp32 and the two products by the scales round by 2^-24 each, the softcap's division,
tanhf (2 ulp, that is 2^-22) and product by 2^-24, 4 x 2^-24 and 2^-24, and a relative change of tanh's argument
changes the result by no more than itself: 3 or 9 x 2^-24 in all, 10 x 2^-24 with the second-order
terms, and half a step of the output type."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diskllm_b200 import capi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def ref_quantize(x, norm=False, norm_w=None, eps=1e-6, add_one=False):
    y = x.detach().cpu().double().numpy()
    if norm:
        y = y / np.sqrt(np.mean(y * y, axis=1, keepdims=True) + float(np.float32(eps)))
        if norm_w is not None:
            y = y * (norm_w.cpu().double().numpy() + (1.0 if add_one else 0.0))
    fine = np.isfinite(y).all(axis=1)
    big = np.abs(np.where(fine[:, None], y, 0.0)).max(axis=1)
    s = (big / 127.0).astype(np.float32)
    s[s < np.finfo(np.float32).tiny] = 0
    d = np.where(s > 0, s, 1).astype(np.float64)
    q = np.where(((s > 0) & fine)[:, None], np.rint(np.where(fine[:, None], y, 0.0) / d[:, None]), 0).astype(np.int8)
    return q, np.where(fine, s, np.float32(np.nan))


def ref_matmul(a, sa, b, sb, softcap=0.0):
    acc = (a.cpu().double() @ b.cpu().double().T).numpy()
    y = acc * sa.cpu().double().numpy()[:, None] * sb.cpu().double().numpy()[None, :]
    return softcap * np.tanh(y / softcap) if softcap > 0 else y


def check_product(got, ref, out_dtype):
    rel = 10 * U + (0 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2 * 1.01)
    g = got.cpu().double().numpy()
    # below the smallest normal number a rounding is absolute
    tiny = float(torch.finfo(out_dtype).tiny)
    big = float(torch.finfo(out_dtype).max)
    inside = np.abs(ref) < big
    bad = inside & (np.abs(g - ref) > rel * np.abs(ref) + rel * tiny)
    assert not bad.any(), (np.argwhere(bad)[:5], g[bad][:5], ref[bad][:5])


def codes(rng, rows, cols, lo=-127, hi=127):
    ld = (cols + 15) // 16 * 16
    full = torch.from_numpy(rng.integers(-128, 128, (rows, ld)).astype(np.int8)).to(DEV)  # padding holds numbers too
    full[:, :cols] = torch.from_numpy(rng.integers(lo, hi + 1, (rows, cols)).astype(np.int8)).to(DEV)
    return full[:, :cols]


# ---- codes ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 17), (3, 255), (5, 1000), (2, 2304), (4, 4096), (7, 4097), (2, 8200),
                                       (1, 40000), (300, 64)])
@pytest.mark.parametrize("norm", [None, "plain", "weight", "one"])
def test_quantize(dtype, rows, cols, norm):
    rng = np.random.default_rng(rows * 7 + cols)
    x = torch.from_numpy((rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1)))).astype(np.float32))
    x = x.to(dtype).to(DEV)
    kw = {}
    if norm:
        kw = dict(norm=True, eps=1e-5, add_one=norm == "one")
        if norm != "plain":
            kw["norm_w"] = torch.from_numpy((1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)).to(DEV)
    q, s = capi.quantize_rows_i8(x, **kw)
    rq, rs = ref_quantize(x, **kw)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,base,stride", [(100, 1, 101), (33, 3, 48), (256, 2, 257), (4096, 1, 4099)])
def test_quantize_strides(dtype, cols, base, stride):
    rng = np.random.default_rng(cols)
    buf = torch.from_numpy(rng.standard_normal(base + 5 * stride).astype(np.float32)).to(dtype).to(DEV)
    x = buf[base:].as_strided((5, cols), (stride, 1))
    ld = (cols + 15) // 16 * 16 + 32
    store = torch.full((6, ld), 77, dtype=torch.int8, device=DEV)
    q, s = capi.quantize_rows_i8(x, q=store[:5, :cols])
    rq, rs = ref_quantize(x)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    assert (store[:, cols:] == 77).all() and (store[5] == 77).all()  # around the rows nothing is written


def test_quantize_ties_and_edges():
    x = torch.zeros(9, 40)
    x[0, :6] = torch.tensor([127.0, 0.5, 1.5, -2.5, -0.5, 126.5])             # scale 1: ties to even
    x[1, :4] = torch.tensor([381.0, 4.5, -7.5, 1.5])                          # scale 3
    x[2, 3] = -5.0                                                            # one value, negative
    # x[3] stays zero
    x[4, :3] = torch.tensor([1e-38, -1e-38, 5e-39])                           # scale below the smallest normal number
    x[5, :2] = torch.tensor([1.5e-36, 1.4e-36])                               # just above it
    x[6, 7], x[7, 8] = float("inf"), float("nan")
    x[8, :3] = torch.tensor([3.4028235e38, -3.4028235e38, 1e38])
    q, s = capi.quantize_rows_i8(x.to(DEV))
    rq, rs = ref_quantize(x)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    assert q[0, :6].tolist() == [127, 0, 2, -2, 0, 126] and q[1, :4].tolist() == [127, 2, -2, 0]
    assert s[3] == 0 and s[4] == 0 and torch.isnan(s[6]) and torch.isnan(s[7])
    q, s = capi.quantize_rows_i8(x[3:4].to(DEV), norm=True, eps=0.0)          # 0 / 0
    assert torch.isnan(s).all() and (q == 0).all()


def test_quantize_no_rows():
    q, s = capi.quantize_rows_i8(torch.empty(0, 20, device=DEV))
    assert q.shape == (0, 20) and s.shape == (0,)


# ---- product -------------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 130, 16), (2, 127, 100), (5, 257, 33), (8, 128, 128), (16, 1000, 129), (17, 300, 640),
         (31, 64, 2304), (33, 129, 255), (64, 512, 4096), (100, 333, 1000), (128, 200, 512), (129, 100, 96),
         (200, 384, 1030), (256, 256, 384), (257, 131, 70), (300, 1111, 600), (513, 520, 200), (3, 20000, 64),
         # several tiles for every SM, whole and ragged in both directions, short and long k
         (512, 19000, 160), (400, 25025, 33), (1001, 9999, 300), (2048, 4736, 96), (3001, 4097, 640), (700, 13000, 2050)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype,cap", [(torch.float32, 0.0), (torch.float32, 30.0), (torch.bfloat16, 0.0),
                                       (torch.float16, 5.0)])
def test_matmul(m, n, k, dtype, cap):
    rng = np.random.default_rng(m * 131 + n * 17 + k)
    a, b = codes(rng, m, k), codes(rng, n, k)
    sa = torch.from_numpy((rng.random(m) * 0.05 + 0.001).astype(np.float32)).to(DEV)
    sb = torch.from_numpy((rng.random(n) * 0.01 + 0.0001).astype(np.float32)).to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = capi.matmul_i8(a, sa, b, sb, softcap=cap, out_dtype=dtype, status=status)
    check_product(got, ref_matmul(a, sa, b, sb, cap), dtype)
    assert status.item() == 0


@pytest.mark.parametrize("k", [1, 15, 31, 4097, 131071])
def test_matmul_extreme_codes(k):
    """all codes -128: sums up to 2^31 - 16384, where a wrong width would show"""
    a = torch.full((3, (k + 15) // 16 * 16), -128, dtype=torch.int8, device=DEV)[:, :k]
    b = torch.full((150, (k + 15) // 16 * 16), -128, dtype=torch.int8, device=DEV)[:, :k]
    one = torch.ones(150, device=DEV)
    got = capi.matmul_i8(a, one[:3], b, one)
    assert (got == float(np.float32(16384 * k))).all()
    b.add_(1).neg_()  # 127, in the same rows
    assert (capi.matmul_i8(a, one[:3], b, one) == float(np.float32(-128 * 127 * k))).all()


def test_matmul_strided_operands_and_output():
    rng = np.random.default_rng(3)
    m, n, k = 19, 150, 90
    big_a, big_b = codes(rng, m, 320), codes(rng, 2 * n, 160)
    a, b = big_a[:, 64:64 + k], big_b[::2, 16:16 + k]  # other columns and rows lie between
    sa, sb = torch.rand(m, device=DEV), torch.rand(n, device=DEV)
    for dtype in TYPES:
        store = torch.full((m + 1, n + 7), 3.0, dtype=dtype, device=DEV)
        out = capi.matmul_i8(a, sa, b, sb, softcap=9.0, out=store[:m, 2:2 + n])
        check_product(out, ref_matmul(a, sa, b, sb, 9.0), dtype)
        assert (store[:, :2] == 3).all() and (store[:, 2 + n:] == 3).all() and (store[m] == 3).all()


def test_matmul_scales():
    """zero, NaN and huge scales reach the rows and columns that they belong to, and no others"""
    rng = np.random.default_rng(4)
    a, b = codes(rng, 20, 64), codes(rng, 140, 64)
    sa, sb = torch.ones(20, device=DEV), torch.ones(140, device=DEV)
    sa[3], sa[7], sb[130] = 0.0, float("nan"), float("inf")
    got = capi.matmul_i8(a, sa, b, sb)
    ref = torch.from_numpy(a.cpu().numpy().astype(np.float64) @ b.cpu().numpy().astype(np.float64).T).float().to(DEV)
    ref = ref * sa[:, None] * sb[None, :]
    assert torch.isnan(got[7]).all() and (got[3, :130] == 0).all() and torch.isnan(got[3, 130])
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(ref, nan=7.0))


def test_matmul_nothing():
    z = torch.empty(0, 32, dtype=torch.int8, device=DEV)
    b, s = torch.ones(5, 32, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)
    assert capi.matmul_i8(z, s[:0], b, s).shape == (0, 5)
    assert capi.matmul_i8(b, s, z, s[:0]).shape == (5, 0)


def test_matmul_repeats_bit_for_bit():
    rng = np.random.default_rng(5)
    a, b = codes(rng, 40, 2000), codes(rng, 700, 2000)
    sa, sb = torch.rand(40, device=DEV), torch.rand(700, device=DEV)
    first = capi.matmul_i8(a, sa, b, sb, softcap=20.0)
    for _ in range(3):
        assert torch.equal(first, capi.matmul_i8(a, sa, b, sb, softcap=20.0))
    one_by_one = torch.cat([capi.matmul_i8(a[i:i + 1], sa[i:i + 1], b, sb, softcap=20.0) for i in range(40)])
    assert torch.equal(first, one_by_one)  # a row's result does not depend on the rows around it


# ---- LM head -------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,hidden,vocab,norm,add_one,cap", [
    (1, 4096, 5000, True, False, 0.0), (3, 2304, 1003, True, True, 30.0), (8, 1000, 777, False, False, 0.0),
    (33, 264, 129, True, False, 15.0), (1, 5, 3, True, True, 0.0),
])
def test_lmhead(rows, hidden, vocab, norm, add_one, cap):
    rng = np.random.default_rng(hidden)
    h = torch.from_numpy((3 * rng.standard_normal((rows, hidden))).astype(np.float32)).to(DEV)
    w = torch.from_numpy((0.05 * rng.standard_normal((vocab, hidden))).astype(np.float32)).to(DEV)
    nw = torch.from_numpy((0.2 * rng.standard_normal(hidden) + (0 if add_one else 1)).astype(np.float32)).to(DEV)
    nw = nw if norm else None
    wq, sw = capi.quantize_rows_i8(w)
    got = capi.lmhead_logits_i8(h, wq, sw, norm_w=nw, add_one=add_one, softcap=cap)
    q, s = ref_quantize(h, True, nw, 1e-6, add_one)
    ref = ref_matmul(torch.from_numpy(q), torch.from_numpy(s), wq, sw, cap)
    check_product(got, ref, torch.float32)


def test_lmhead_is_near_the_unquantised_one():
    """Rounding to codes moves each product's factors by at most half a scale: with row maxima of
    about 4 sigma that is a relative error near 1 % of the logits' standard deviation."""
    rng = np.random.default_rng(11)
    h = torch.from_numpy(rng.standard_normal((4, 2048)).astype(np.float32)).to(DEV)
    w = torch.from_numpy((0.05 * rng.standard_normal((3000, 2048))).astype(np.float32)).to(DEV)
    full = capi.lmhead_logits(h, w)
    low = capi.lmhead_logits_i8(h, *capi.quantize_rows_i8(w))
    # each code is off by at most 1/2 (uniform: variance 1/12 of a scale); both factors: two such errors
    step = (w.abs().amax(1) / 127).pow(2).mean() / w.pow(2).mean() + (h.abs().amax(1) / 127).pow(2).mean() / h.pow(2).mean()
    expected = (step / 12).sqrt() * full.std()
    assert (low - full).std() < 2 * expected


def test_lmhead_feeds_the_sampler():
    rng = np.random.default_rng(12)
    h = torch.from_numpy(rng.standard_normal((6, 512)).astype(np.float32)).to(DEV)
    wq, sw = capi.quantize_rows_i8(torch.from_numpy(rng.standard_normal((4000, 512)).astype(np.float32)).to(DEV))
    lg = capi.lmhead_logits_i8(h, wq, sw)
    tok = capi.sample_batch(lg, torch.zeros(6, device=DEV), dict(temperature=0.0))
    assert torch.equal(tok.long(), lg.argmax(1))


def test_lmhead_graph_and_streams():
    """a captured call (workspace of its own) replays on new inputs; calls on two streams at once"""
    rng = np.random.default_rng(13)
    wq, sw = capi.quantize_rows_i8(torch.from_numpy(rng.standard_normal((2000, 640)).astype(np.float32)).to(DEV))
    hs = [torch.from_numpy(rng.standard_normal((5, 640)).astype(np.float32)).to(DEV) for _ in range(4)]
    refs = [capi.lmhead_logits_i8(h, wq, sw) for h in hs]
    h, out = hs[0].clone(), torch.empty(5, 2000, device=DEV)
    ws = torch.empty(1 << 16, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        capi.lmhead_logits_i8(h, wq, sw, logits=out, workspace=ws)
    for i in (2, 1, 3):
        h.copy_(hs[i])
        g.replay()
        assert torch.equal(out, refs[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(capi.lmhead_logits_i8(hs[i], wq, sw))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, refs[i]) for o in outs[i])


def test_capture_without_a_workspace_is_refused():
    lib = capi.load_library()
    h, sw = torch.zeros(2, 64, device=DEV), torch.ones(32, device=DEV)
    w, out = torch.zeros(32, 64, dtype=torch.int8, device=DEV), torch.zeros(2, 32, device=DEV)

    def call():
        return lib.dllm_cuda_lmhead_logits_i8(2, 64, 32, h.data_ptr(), None, 1e-6, 0, w.data_ptr(), 64, sw.data_ptr(), 0.0,
                                              out.data_ptr(), None, None, 0, torch.cuda.current_stream().cuda_stream)

    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out.add_(1)
        rc = call()
    assert rc == capi.DLLM_ERR_INVALID_ARG
    g.replay()
    assert (out == 1).all()
    assert call() == capi.DLLM_OK  # outside a capture the library's own buffer serves
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("m,n,k", [(16, 4096, 4096), (300, 30000, 640), (1, 40000, 256)])
def test_a_wait_that_runs_out_is_reported(m, n, k):
    """the product's issuing threads wait for something that nothing completes (no copy or product is in
    flight to it): the kernel returns within a moment with DLLM_ROW_ERR_TIMEOUT, and the next call is right"""
    import time

    rng = np.random.default_rng(m)
    a, b = codes(rng, m, k), codes(rng, n, k)
    sa, sb = torch.rand(m, device=DEV), torch.rand(n, device=DEV)
    want = capi.matmul_i8(a, sa, b, sb)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    capi.inject_wait_timeout(capi.FAULT_PRODUCT_WAIT, 1000)
    try:
        start = time.time()
        capi.matmul_i8(a, sa, b, sb, status=status)
        torch.cuda.synchronize()
        assert time.time() - start < 2.0
    finally:
        capi.inject_wait_timeout(capi.FAULT_NONE)
    assert status.item() == capi.ROW_ERR_TIMEOUT
    status.zero_()
    for _ in range(3):
        assert torch.equal(capi.matmul_i8(a, sa, b, sb, status=status), want)
    assert status.item() == 0


def test_tensor_refusals():
    q = torch.zeros(4, 40, dtype=torch.int8, device=DEV)
    s = torch.ones(4, device=DEV)
    good = torch.zeros(4, 48, dtype=torch.int8, device=DEV)[:, :40]
    x = torch.zeros(4, 40, device=DEV)
    for call in (
        lambda: capi.matmul_i8(q, s, good, s),                       # rows of 40 bytes
        lambda: capi.matmul_i8(good, s, good[:, 1:], s),             # another k
        lambda: capi.matmul_i8(good[:, 1:], s, good[:, 1:], s),      # base off 16 bytes
        lambda: capi.matmul_i8(good, s[:3], good, s),
        lambda: capi.matmul_i8(good, s.double(), good, s),
        lambda: capi.matmul_i8(good, s, good, s, out_dtype=torch.float64),
        lambda: capi.matmul_i8(good.cpu(), s, good, s),
        lambda: capi.matmul_i8(good, s, good.cpu(), s),
        lambda: capi.matmul_i8(x, s, good, s),
        lambda: capi.matmul_i8(good, s, good, s, softcap=-1.0),
        lambda: capi.quantize_rows_i8(x.t()),
        lambda: capi.quantize_rows_i8(x.double()),
        lambda: capi.quantize_rows_i8(x.cpu()),
        lambda: capi.quantize_rows_i8(x, norm_w=torch.ones(40, device=DEV)),
        lambda: capi.quantize_rows_i8(x, norm=True, norm_w=torch.ones(39, device=DEV)),
        lambda: capi.quantize_rows_i8(x, q=q),
        lambda: capi.lmhead_logits_i8(x, good[:, :32], s),
        lambda: capi.lmhead_logits_i8(x.half(), good, s),
        lambda: capi.lmhead_logits_i8(x, good, s, workspace=torch.empty(64, dtype=torch.uint8, device=DEV)),
    ):
        with pytest.raises(capi.DllmError):
            call()


# ---- numbers below the smallest normal one --------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [40, 1000, 4096, 10001, 20000])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-6])
def test_quantize_rows_of_subnormal_values(dtype, cols, eps):
    rng = np.random.default_rng(cols)
    bits = 22 if dtype == torch.float32 else 6  # of the subnormal numbers' 23 and 7
    ints = rng.integers(-(1 << bits), 1 << bits, (3, cols)).astype(np.float64)
    x = torch.from_numpy(np.ldexp(ints, -149 if dtype == torch.float32 else -133).astype(np.float32)).to(dtype).to(DEV)
    q, s = capi.quantize_rows_i8(x, norm=True, eps=eps)
    rq, rs = ref_quantize(x, norm=True, eps=eps)
    assert eps == 1e-40 or (rs > 0).all()
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.parametrize("cols", [16384, 40000])
def test_quantize_subnormal_weights(cols):
    x = torch.full((2, cols), 2.0 ** -30, device=DEV)
    x[0, 5], x[1, 7] = 3.0, -2.0
    w = torch.full((cols,), float(np.ldexp(8388607.0, -149)), device=DEV)
    q, s = capi.quantize_rows_i8(x, norm=True, norm_w=w)
    rq, rs = ref_quantize(x, norm=True, norm_w=w)
    assert (rs > 0).all()
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.parametrize("m,n,k", [(5, 257, 33), (3, 20000, 64)])
def test_matmul_subnormal_results(m, n, k):
    """the products by the scales round to multiples of 2^-149, half a step each: the first's is multiplied by
    b_scale <= 1, so the two make at most a step"""
    rng = np.random.default_rng(n)
    a, b = codes(rng, m, k), codes(rng, n, k)
    sa = torch.from_numpy(np.ldexp(rng.random(m) + 0.5, -135).astype(np.float32)).to(DEV)
    sb = torch.from_numpy(np.ldexp(rng.random(n) + 0.5, -8).astype(np.float32)).to(DEV)
    got = capi.matmul_i8(a, sa, b, sb).cpu().double().numpy()
    ref = ref_matmul(a, sa, b, sb)
    assert ((np.abs(ref) < 2.0 ** -126) & (np.abs(ref) > 2.0 ** -140)).mean() > 0.9
    assert (np.abs(got - ref) <= 3 * U * np.abs(ref) + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [40, 1000, 4096, 20000])
def test_quantize_subnormal_values_beside_a_normal_one(dtype, cols):
    """the scale is just above the smallest normal number, so the subnormal values have codes of -1, 0 and 1"""
    rng = np.random.default_rng(cols)
    ints = rng.integers(-127, 128, (2, cols)).astype(np.float64)
    ints[:, cols // 3] = [128 * 127.0, 128 * 129.0]
    x = torch.from_numpy(np.ldexp(ints, -133).astype(np.float32)).to(dtype).to(DEV)
    q, s = capi.quantize_rows_i8(x)
    rq, rs = ref_quantize(x)
    assert (rs > 0).all() and (np.abs(rq) == 1).any()
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
