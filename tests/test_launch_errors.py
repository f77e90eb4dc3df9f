"""What the int8 and beam calls report when CUDA fails: the error itself, and nothing that an earlier
failure left behind."""
import ctypes as C

import pytest
import torch

from diskllm_b200 import capi
from test_int8_beam_args import _beam, _lmhead, _matmul, _quantize, _reorder

ERR_CUDA = 3
CALLS = dict(quantize=_quantize, matmul=_matmul, lmhead=_lmhead, reorder=_reorder,
             select=lambda **kw: capi.load_library().dllm_cuda_beam_select(C.byref(_beam(**kw)), None))


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine on which every launch fails")
@pytest.mark.parametrize("name", CALLS)
def test_a_failed_launch_names_its_error(name):
    """without a GPU no launch succeeds (the arguments are placeholders that nothing reads)"""
    lib = capi.load_library()
    assert _quantize(rows=-1) == capi.DLLM_ERR_INVALID_ARG
    before = lib.dllm_cuda_last_error()
    assert CALLS[name]() == ERR_CUDA
    message = lib.dllm_cuda_last_error()
    assert message and message != before and b"no error" not in message, message


@pytest.mark.gpu
def test_a_refused_launch_names_its_error():
    """a stream whose capture has become invalid takes no launches until the capture ends; the calls say so, and
    work again afterwards"""
    dev = torch.device("cuda", 0)
    lib, rt = capi.load_library(), C.CDLL("libcudart.so.12")
    x, sc = torch.zeros(4, 100, device=dev), torch.zeros(1, 4, device=dev)
    q, scale = torch.ones(4, 112, dtype=torch.int8, device=dev), torch.ones(4, device=dev)
    out, ws = torch.zeros(4, 4, device=dev), torch.empty(1 << 16, dtype=torch.uint8, device=dev)
    desc, best = capi.fill_beam_desc(x, sc, 4, workspace=ws)
    parents = torch.tensor([[1, 0, 3, 2]], dtype=torch.int32, device=dev)
    state = torch.arange(4, dtype=torch.float32, device=dev)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    s = C.c_void_p(stream.cuda_stream)
    calls = dict(
        quantize=lambda: lib.dllm_cuda_quantize_rows_i8(4, 100, x.data_ptr(), 100, 0, 0, None, 0.0, 0, q.data_ptr(), 112,
                                                        scale.data_ptr(), s),
        matmul=lambda: lib.dllm_cuda_matmul_i8(4, 4, 100, q.data_ptr(), 112, scale.data_ptr(), q.data_ptr(), 112,
                                               scale.data_ptr(), 0.0, out.data_ptr(), 4, 0, None, s),
        lmhead=lambda: lib.dllm_cuda_lmhead_logits_i8(4, 100, 4, x.data_ptr(), None, 1e-6, 0, q.data_ptr(), 112,
                                                      scale.data_ptr(), 0.0, out.data_ptr(), None, ws.data_ptr(),
                                                      ws.numel(), s),
        select=lambda: lib.dllm_cuda_beam_select(C.byref(desc), s),
        reorder=lambda: lib.dllm_cuda_beam_reorder(1, 4, parents.data_ptr(), 1, (C.c_void_p * 1)(state.data_ptr()), 4, 1, 0,
                                                   4, s),
        without_scratch=lambda: lib.dllm_cuda_lmhead_logits_i8(4, 100, 4, x.data_ptr(), None, 1e-6, 0, q.data_ptr(), 112,
                                                               scale.data_ptr(), 0.0, out.data_ptr(), None, None, 0, s))
    graph = C.c_void_p()
    assert rt.cudaStreamBeginCapture(s, 2) == 0
    try:
        assert rt.cudaStreamSynchronize(s) != 0  # not allowed in a capture, which is invalid from here on
        for name, call in calls.items():
            rc, message = call(), lib.dllm_cuda_last_error()
            if name == "without_scratch":
                assert rc == capi.DLLM_ERR_INVALID_ARG and b"workspace" in message
            else:
                assert rc == ERR_CUDA and b"captur" in message, (name, rc, message)
    finally:
        assert rt.cudaStreamEndCapture(s, C.byref(graph)) != 0 and not graph
        rt.cudaGetLastError()
    for name, call in calls.items():
        assert call() == capi.DLLM_OK, name
    torch.cuda.synchronize()
    assert state.tolist() == [1.0, 0.0, 3.0, 2.0] and best[2].tolist() == [[0, 1, 2, 3]]


@pytest.mark.gpu
def test_a_failed_allocation_does_not_fail_the_next_call():
    """out of memory for the library's scratch, then the same call with the caller's"""
    dev = torch.device("cuda", 0)
    lib = capi.load_library()
    h, sw = torch.ones(3, 64, device=dev), torch.ones(32, device=dev)
    w, out = torch.ones(32, 64, dtype=torch.int8, device=dev), torch.zeros(3, 32, device=dev)
    ws = torch.empty(4096, dtype=torch.uint8, device=dev)
    x, sc = torch.zeros(4, 100, device=dev), torch.zeros(1, 4, device=dev)
    desc, best = capi.fill_beam_desc(x, sc, 4)
    stream = torch.cuda.Stream()  # a stream that the library has no scratch for yet
    beam_ws = torch.empty(1 << 16, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()

    def head(ptr, size):
        return lib.dllm_cuda_lmhead_logits_i8(3, 64, 32, h.data_ptr(), None, 1e-6, 0, w.data_ptr(), 64, sw.data_ptr(), 0.0,
                                              out.data_ptr(), None, ptr, size, stream.cuda_stream)

    def select():
        return lib.dllm_cuda_beam_select(C.byref(desc), stream.cuda_stream)

    capi.fail_allocations(2)
    try:
        assert head(None, 0) == capi.DLLM_ERR_OOM and b"scratch" in lib.dllm_cuda_last_error()
        assert head(ws.data_ptr(), 4096) == capi.DLLM_OK
        assert select() == capi.DLLM_ERR_OOM
        desc.workspace, desc.workspace_bytes = beam_ws.data_ptr(), beam_ws.numel()
        assert select() == capi.DLLM_OK
    finally:
        capi.fail_allocations(0)
    torch.cuda.synchronize()
    # codes of 127 with a scale of 1 / 127 x 1 / sqrt(1 + 1e-6): 64 less 3.2e-5, and 3 roundings of 64 x 2^-24
    assert (out - 64).abs().max() < 1e-4 and best[2].tolist() == [[0, 1, 2, 3]]


@pytest.mark.gpu
def test_scratch_cannot_grow_during_another_streams_capture():
    """the call is refused, and the scratch that was there serves again"""
    dev = torch.device("cuda", 0)
    lib, rt = capi.load_library(), C.CDLL("libcudart.so.12")
    w, sw = torch.ones(32, 64, dtype=torch.int8, device=dev), torch.ones(32, device=dev)
    h, out = torch.ones(2000, 64, device=dev), torch.zeros(2000, 32, device=dev)
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def head(rows):
        return lib.dllm_cuda_lmhead_logits_i8(rows, 64, 32, h.data_ptr(), None, 1e-6, 0, w.data_ptr(), 64, sw.data_ptr(), 0.0,
                                              out.data_ptr(), None, None, 0, stream.cuda_stream)

    assert head(3) == capi.DLLM_OK
    torch.cuda.synchronize()
    graph = C.c_void_p()
    assert rt.cudaStreamBeginCapture(C.c_void_p(other.cuda_stream), 0) == 0
    try:
        assert head(2000) == capi.DLLM_ERR_OOM
        assert head(3) == capi.DLLM_OK
    finally:
        rt.cudaStreamEndCapture(C.c_void_p(other.cuda_stream), C.byref(graph))
        rt.cudaGetLastError()
    torch.cuda.synchronize()
    out.zero_()
    assert head(2000) == capi.DLLM_OK
    torch.cuda.synchronize()
    assert (out - 64).abs().max() < 1e-4
