"""Host threads that call the C entry points at once with the library's own scratch (workspace NULL): on one
stream, where the kernels of two calls must not alternate and a buffer must not be freed while another
call is about to use it, and on cudaStreamPerThread, one handle for a stream of every thread."""
from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest
import torch

from diskllm_b200 import capi
from test_gpu_beam import beam_scores, rows
from util import u24

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
PER_THREAD = 2  # the handle cudaStreamPerThread


class Head:
    """LM heads of growing sizes: each needs more scratch than the one before"""

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        wq, sw = capi.quantize_rows_i8(torch.from_numpy(rng.standard_normal((700 + seed, 640)).astype(np.float32)).to(DEV))
        hs = [torch.from_numpy(rng.standard_normal((n + seed, 640)).astype(np.float32)).to(DEV) for n in (1, 9, 40, 200)]
        self.cases = [(h, wq, sw, torch.empty(h.shape[0], wq.shape[0], device=DEV)) for h in hs]
        self.want = [capi.lmhead_logits_i8(h, wq, sw) for h in hs]

    def call(self, i, stream):
        h, wq, sw, out = self.cases[i]
        return capi.load_library().dllm_cuda_lmhead_logits_i8(
            h.shape[0], 640, wq.shape[0], h.data_ptr(), None, 1e-6, 0, wq.data_ptr(), 640, sw.data_ptr(), 0.0,
            out.data_ptr(), None, None, 0, stream)

    def wrong(self, i):
        return not torch.equal(self.cases[i][3], self.want[i])


class Select:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.cases, self.want = [], []
        for n in (1, 4, 12, 30):
            x, sc = rows(rng, 4 * (n + seed), 9000, torch.float32), beam_scores(rng, n + seed, 4)
            d, out = capi.fill_beam_desc(x, sc, 8)
            self.cases.append((d, out, x, sc))
            self.want.append(capi.beam_select(x, sc, 8))

    def call(self, i, stream):
        return capi.load_library().dllm_cuda_beam_select(C.byref(self.cases[i][0]), stream)

    def wrong(self, i):
        return not all(torch.equal(a, b) for a, b in zip(self.cases[i][1], self.want[i]))


class Sample:
    P = dict(temperature=0.8, top_k=40, top_p=0.95)

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.cases, self.want = [], []
        for n in (1, 6, 20, 70):
            x = rows(rng, n + seed, 9000, torch.float32)
            u = torch.from_numpy(u24(rng, n + seed)).to(DEV)
            tok = torch.empty(n + seed, dtype=torch.int32, device=DEV)
            self.cases.append((x, u, tok))
            self.want.append(capi.sample_batch(x, u, self.P))

    def call(self, i, stream):
        x, u, tok = self.cases[i]
        capi.sample_batch(x, u, self.P, token=tok, stream=stream)
        return capi.DLLM_OK

    def wrong(self, i):
        return not torch.equal(self.cases[i][2], self.want[i])


def run(works, stream, rounds):
    """every work in a thread of its own, all starting together; the number of wrong results"""
    rcs, start = [], threading.Barrier(len(works))

    def go(w):
        start.wait()
        for r in range(rounds):
            for i in range(4):
                rcs.append(w.call(i, stream))

    threads = [threading.Thread(target=go, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert rcs == [capi.DLLM_OK] * (4 * rounds * len(works))
    return sum(w.wrong(i) for w in works for i in range(4))


@pytest.mark.parametrize("kinds", [(Head,) * 4, (Select,) * 4, (Head, Select, Sample, Head, Select, Sample)])
def test_threads_on_one_stream(kinds):
    works = [k(seed) for seed, k in enumerate(kinds)]
    for _ in range(3):
        stream = torch.cuda.Stream()  # whose buffer grows while the threads call
        torch.cuda.synchronize()
        assert run(works, stream.cuda_stream, 20) == 0


@pytest.mark.parametrize("kinds", [(Head,) * 4, (Select,) * 4, (Head, Select, Sample, Head, Select, Sample)])
def test_threads_on_their_own_default_streams(kinds):
    works = [k(seed) for seed, k in enumerate(kinds)]
    torch.cuda.synchronize()
    for _ in range(5):  # new threads each time: they take over the ended ones' buffers
        assert run(works, PER_THREAD, 8) == 0
