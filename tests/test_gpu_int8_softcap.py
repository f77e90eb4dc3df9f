"""The softcap of the int8 product at the ends of its range."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from test_gpu_int8 import DEV, check_product, codes, ref_matmul

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [64, 2048])
def test_softcap_at_the_ends_of_its_range(k):
    """a channel's b_scale / softcap above the largest number: sums of 0 stay 0, the others reach the cap"""
    a, b = codes(np.random.default_rng(1), 20, k), codes(np.random.default_rng(2), 300, k)
    a[3], b[7] = 0, 0
    sa, sb = torch.full((20,), 0.5, device=DEV), torch.full((300,), 8.0, device=DEV)
    sb[9] = float("nan")
    tiny = float(np.finfo(np.float32).tiny)
    for cap in (tiny, 1e-37, 1e30, 3.3e38):
        got = capi.matmul_i8(a, sa, b, sb, softcap=cap)
        assert torch.isnan(got[:, 9]).all()
        ref = ref_matmul(a, sa, b, sb, float(np.float32(cap)))
        keep = [j for j in range(300) if j != 9]
        assert torch.isfinite(got[:, keep]).all()
        check_product(got[:, keep], ref[:, keep], torch.float32)


@pytest.mark.parametrize("cap", [1e-38, 1e-45])
def test_softcap_below_the_smallest_normal_number_is_refused(cap):
    a, s = torch.zeros(4, 16, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    with pytest.raises(capi.DllmError):
        capi.matmul_i8(a, s, a, s, softcap=cap)
    with pytest.raises(capi.DllmError):
        capi.lmhead_logits_i8(torch.zeros(2, 16, device=DEV), a, s, softcap=cap)
