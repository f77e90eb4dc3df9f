"""The int8 LM head at the sizes that serve weights and batches: rows by the hundred, whose codes are made
by other kernels than a few rows', and products in which every SM takes several tiles while the codes are
still being made.  Definitions and tolerances are those of test_gpu_int8."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from test_gpu_int8 import DEV, TYPES, check_product, ref_matmul, ref_quantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("rows,cols", [(150, 512), (150, 513), (148, 1023), (147, 1024), (160, 1024), (200, 1025),
                                       (148, 2048), (149, 2304), (160, 4096), (160, 4097), (150, 8191), (148, 8192),
                                       (149, 8193), (150, 16385)])
@pytest.mark.parametrize("norm", [None, "plain", "weight", "one"])
def test_quantize_many_rows(dtype, aligned, rows, cols, norm):
    rng = np.random.default_rng(rows * 7 + cols)
    stride = (cols + 15) // 16 * 16 + (0 if aligned else 1)
    store = torch.from_numpy((rng.standard_normal((rows, stride)) * np.exp(rng.standard_normal((rows, 1)))).astype(np.float32))
    x = store.to(dtype).to(DEV)[:, :cols]
    x[7], x[rows - 1, cols - 1], x[rows - 2, cols // 2] = 0.0, float("nan"), float("inf")
    kw = {}
    if norm:
        kw = dict(norm=True, eps=1e-5, add_one=norm == "one")
        if norm != "plain":
            kw["norm_w"] = torch.from_numpy((1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)).to(DEV)
    ld = (cols + 15) // 16 * 16 + 16
    out = torch.full((rows + 1, ld), 77, dtype=torch.int8, device=DEV)
    q, s = capi.quantize_rows_i8(x, q=out[:rows, :cols], **kw)
    with np.errstate(invalid="ignore"):
        rq, rs = ref_quantize(x, **kw)
    np.testing.assert_array_equal(s.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    assert (out[:, cols:] == 77).all() and (out[rows] == 77).all()  # around the rows nothing is written


@pytest.mark.parametrize("rows", [1, 40, 200, 300])
@pytest.mark.parametrize("hidden,vocab,add_one,cap", [(200, 40000, False, 0.0), (96, 60001, True, 20.0),
                                                      (2304, 19500, True, 30.0)])
def test_lmhead_of_many_tiles(rows, hidden, vocab, add_one, cap):
    """a CTA of the product takes several tiles, with fewer blocks of k than stages or with more; up to 300 rows"""
    rng = np.random.default_rng(hidden + rows)
    h = torch.from_numpy((3 * rng.standard_normal((rows, hidden))).astype(np.float32)).to(DEV)
    w = torch.from_numpy((0.05 * rng.standard_normal((vocab, hidden))).astype(np.float32)).to(DEV)
    nw = torch.from_numpy((0.2 * rng.standard_normal(hidden) + (0 if add_one else 1)).astype(np.float32)).to(DEV)
    wq, sw = capi.quantize_rows_i8(w)
    rq, rs = ref_quantize(w)
    np.testing.assert_array_equal(sw.cpu().numpy(), rs)
    np.testing.assert_array_equal(wq.cpu().numpy(), rq)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = [capi.lmhead_logits_i8(h, wq, sw, norm_w=nw, add_one=add_one, softcap=cap, status=status) for _ in range(3)]
    q, s = ref_quantize(h, True, nw, 1e-6, add_one)
    check_product(got[0], ref_matmul(torch.from_numpy(q), torch.from_numpy(s), wq, sw, cap), torch.float32)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and status.item() == 0


def test_lmhead_right_after_the_weights_codes():
    """no pause between making the weights' codes, in the same buffers, and the product that reads them"""
    rng = np.random.default_rng(6)
    h = torch.from_numpy(rng.standard_normal((20, 512)).astype(np.float32)).to(DEV)
    ws = [torch.from_numpy(rng.standard_normal((30000, 512)).astype(np.float32)).to(DEV) for _ in range(3)]
    want = [capi.lmhead_logits_i8(h, *capi.quantize_rows_i8(w)) for w in ws]
    q, s = capi.quantize_rows_i8(ws[0])
    got = []
    for w in ws + ws:
        capi.quantize_rows_i8(w, q=q, scale=s)
        got.append(capi.lmhead_logits_i8(h, q, s))
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 3])
