"""ctypes binding of libdiskllm_cuda.so (include/diskllm_cuda.h, include/sampler.h).

This is the Python host side above the C ABI.  It mirrors DiskLLM's sampler interface
(include/sampler.h:7-34: sampler_create / sampler_free / sampler_apply_*_penalty /
sampler_sample / greedy_sample) and adds the batched device entry point.  The library is
required: loading it on a machine without the built .so raises, and nothing here falls back
to a host implementation.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import threading

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libdiskllm_cuda.so")

DLLM_OK = 0
DLLM_ERR_INVALID_ARG = 1
DLLM_ERR_OOM = 2
DLLM_ERR_UNSUPPORTED = 6
STATUS_NAMES = {0: "OK", 1: "INVALID_ARG", 2: "OOM", 3: "CUDA", 4: "NCCL", 5: "TIMEOUT",
                6: "UNSUPPORTED"}
DTYPE_F32 = 0
DTYPE_BF16 = 1
DTYPE_F16 = 2  # output weights, the int8 and the beam calls
BEAM_MAX, BEAM_K_MAX = 128, 256
MODE_TOPP_SORTED = 0x1
MODE_PEN_TRUE_DIV = 0x2
MODE_MINP_RELATIVE = 0x4
ROW_ERR_HIST_TABLE = 1
ROW_ERR_NONFINITE = 2
ROW_ERR_TOPK_LARGE = 4
ROW_ERR_WALK = 8
ROW_ERR_TIMEOUT = 16
ROW_TOPP_EDGE = 32  # information: the index-order top-p cut lies near the threshold

# every symbol the public headers declare
EXPORTS = [
    "dllm_cuda_sample_batch", "dllm_cuda_version", "dllm_cuda_last_error",
    "dllm_cuda_set_debug_counters", "dllm_cuda_workspace_bytes", "dllm_cuda_sample_batch_static",
    "dllm_cuda_set_timing_events", "dllm_cuda_shard_candidates", "dllm_cuda_merge_sample",
    "dllm_cuda_append_history", "dllm_cuda_lmhead_logits",
    "dllm_cuda_quantize_rows_i8", "dllm_cuda_matmul_i8", "dllm_cuda_lmhead_logits_i8",
    "dllm_cuda_lmhead_i8_workspace_bytes", "dllm_cuda_beam_select", "dllm_cuda_beam_workspace_bytes",
    "dllm_cuda_beam_reorder",
    "dllm_cuda_debug_inject_wait_timeout", "dllm_cuda_debug_fail_allocations",
    "dllm_cuda_peer_exchange_create", "dllm_cuda_peer_exchange_open", "dllm_cuda_peer_exchange_close",
    "dllm_cuda_peer_exchange_free", "dllm_cuda_shard_candidates_peer", "dllm_cuda_merge_sample_peer",
    "diskllm_grammar_init_from_file", "diskllm_grammar_init_from_str", "diskllm_grammar_init_json",
    "diskllm_grammar_free", "diskllm_grammar_reset", "diskllm_grammar_accept_str", "diskllm_grammar_advance",
    "diskllm_grammar_is_finished", "diskllm_grammar_apply_mask", "dllm_grammar_build_bitmask",
    "dllm_grammar_vocab_create", "dllm_grammar_vocab_free", "dllm_grammar_build_bitmask_cached",
    "dllm_sampler_get_rng_state", "dllm_sampler_set_rng_state",
    "sampler_create", "sampler_free", "sampler_apply_repetition_penalty",
    "sampler_apply_presence_penalty", "sampler_sample", "greedy_sample",
]


class DllmError(RuntimeError):
    pass


class SamplerParams(C.Structure):
    """dllm_sampler_params"""
    _fields_ = [
        ("temperature", C.c_float),
        ("top_p", C.c_float),
        ("min_p", C.c_float),
        ("top_k", C.c_int),
        ("repetition", C.c_float),
        ("presence", C.c_float),
        ("frequency", C.c_float),
    ]


class SamplerConfig(C.Structure):
    """sampler_config (DiskLLM include/sampler.h:10-16)"""
    _fields_ = [
        ("temperature", C.c_float),
        ("top_k", C.c_int),
        ("top_p", C.c_float),
        ("min_p", C.c_float),
        ("seed", C.c_uint64),
    ]


class BatchDesc(C.Structure):
    """dllm_batch_desc"""
    _fields_ = [
        ("rows", C.c_int),
        ("vocab", C.c_int),
        ("row_stride", C.c_int64),
        ("dtype", C.c_int),
        ("logits", C.c_void_p),
        ("mask", C.c_void_p),
        ("mask_stride", C.c_int64),
        ("hist_ids", C.c_void_p),
        ("hist_off", C.c_void_p),
        ("hist_max", C.c_int),
        ("uniforms", C.c_void_p),
        ("params", SamplerParams),
        ("row_params", C.c_void_p),
        ("topk_max", C.c_int),
        ("flags", C.c_uint),
        ("token", C.c_void_p),
        ("probs", C.c_void_p),
        ("probs_stride", C.c_int64),
        ("pen_logits", C.c_void_p),
        ("pen_stride", C.c_int64),
        ("status", C.c_void_p),
        ("topk_ids", C.c_void_p),
        ("topk_stride", C.c_int64),
        ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_size_t),
    ]


class BeamDesc(C.Structure):
    """dllm_beam_desc"""
    _fields_ = [
        ("batch", C.c_int),
        ("beams", C.c_int),
        ("vocab", C.c_int),
        ("k", C.c_int),
        ("row_stride", C.c_int64),
        ("dtype", C.c_int),
        ("logits", C.c_void_p),
        ("mask", C.c_void_p),
        ("mask_stride", C.c_int64),
        ("scores", C.c_void_p),
        ("finished", C.c_void_p),
        ("eos", C.c_int),
        ("lengths", C.c_void_p),
        ("length_penalty", C.c_float),
        ("out_score", C.c_void_p),
        ("out_parent", C.c_void_p),
        ("out_token", C.c_void_p),
        ("out_finished", C.c_void_p),
        ("out_lengths", C.c_void_p),
        ("status", C.c_void_p),
        ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_size_t),
    ]


_lib = None


def load_library(path: str = LIB_PATH) -> C.CDLL:
    """Loads libdiskllm_cuda.so; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise DllmError(f"{path} is missing: build it with `python -m diskllm_b200.build`")
    lib = C.CDLL(path)
    lib.dllm_cuda_sample_batch.restype = C.c_int
    lib.dllm_cuda_sample_batch.argtypes = [C.POINTER(BatchDesc), C.c_void_p]
    lib.dllm_cuda_set_debug_counters.restype = C.c_int
    lib.dllm_cuda_set_debug_counters.argtypes = [C.c_void_p]
    lib.dllm_cuda_shard_candidates.restype = C.c_int
    lib.dllm_cuda_shard_candidates.argtypes = [C.POINTER(BatchDesc), C.c_int64, C.c_int64, C.c_int,
                                               C.c_void_p, C.c_void_p, C.c_void_p]
    lib.dllm_cuda_merge_sample.restype = C.c_int
    lib.dllm_cuda_merge_sample.argtypes = [C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p,
                                           C.POINTER(SamplerParams), C.c_void_p, C.c_void_p, C.c_void_p,
                                           C.c_void_p, C.c_void_p]
    lib.dllm_cuda_lmhead_logits.restype = C.c_int
    lib.dllm_cuda_lmhead_logits.argtypes = [C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_float, C.c_int,
                                            C.c_void_p, C.c_int, C.c_float, C.c_void_p, C.c_void_p]
    lib.dllm_cuda_append_history.restype = C.c_int
    lib.dllm_cuda_append_history.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    lib.dllm_cuda_set_timing_events.restype = C.c_int
    lib.dllm_cuda_set_timing_events.argtypes = [C.c_void_p, C.c_void_p]
    lib.dllm_cuda_sample_batch_static.restype = C.c_int
    lib.dllm_cuda_sample_batch_static.argtypes = [C.POINTER(BatchDesc), C.c_void_p]
    lib.dllm_cuda_debug_inject_wait_timeout.restype = C.c_int
    lib.dllm_cuda_debug_inject_wait_timeout.argtypes = [C.c_int, C.c_longlong]
    lib.dllm_cuda_debug_fail_allocations.restype = C.c_int
    lib.dllm_cuda_debug_fail_allocations.argtypes = [C.c_int]
    for name, args in (("dllm_cuda_peer_exchange_create", [C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p]),
                       ("dllm_cuda_peer_exchange_open", [C.c_void_p, C.c_void_p]),
                       ("dllm_cuda_peer_exchange_close", [C.c_void_p]),
                       ("dllm_cuda_peer_exchange_free", [C.c_void_p]),
                       ("dllm_cuda_shard_candidates_peer", [C.POINTER(BatchDesc), C.c_int64, C.c_int64, C.c_int,
                                                            C.c_void_p, C.c_int, C.c_int, C.c_uint64, C.c_void_p]),
                       ("dllm_cuda_merge_sample_peer", [C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_uint64,
                                                        C.POINTER(SamplerParams), C.c_void_p, C.c_void_p, C.c_void_p,
                                                        C.c_void_p, C.c_void_p])):
        f = getattr(lib, name)
        f.restype = C.c_int
        f.argtypes = args
    i32, i64, f32, ptr = C.c_int, C.c_int64, C.c_float, C.c_void_p
    for name, args in (("dllm_cuda_quantize_rows_i8", [i32, i32, ptr, i64, i32, i32, ptr, f32, i32, ptr, i64, ptr, ptr]),
                       ("dllm_cuda_matmul_i8", [i32, i32, i32, ptr, i64, ptr, ptr, i64, ptr, f32, ptr, i64, i32, ptr,
                                                ptr]),
                       ("dllm_cuda_lmhead_logits_i8", [i32, i32, i32, ptr, ptr, f32, i32, ptr, i64, ptr, f32, ptr, ptr,
                                                       ptr, C.c_size_t, ptr]),
                       ("dllm_cuda_beam_select", [C.POINTER(BeamDesc), ptr]),
                       ("dllm_cuda_beam_reorder", [i32, i32, ptr, i32, ptr, i64, i32, i64, i64, ptr])):
        f = getattr(lib, name)
        f.restype = C.c_int
        f.argtypes = args
    lib.dllm_cuda_lmhead_i8_workspace_bytes.restype = C.c_size_t
    lib.dllm_cuda_lmhead_i8_workspace_bytes.argtypes = [i32, i32]
    lib.dllm_cuda_beam_workspace_bytes.restype = C.c_size_t
    lib.dllm_cuda_beam_workspace_bytes.argtypes = [C.POINTER(BeamDesc)]
    lib.dllm_cuda_workspace_bytes.restype = C.c_size_t
    lib.dllm_cuda_workspace_bytes.argtypes = [C.POINTER(BatchDesc)]
    lib.dllm_cuda_version.restype = C.c_char_p
    lib.dllm_cuda_last_error.restype = C.c_char_p
    lib.dllm_sampler_get_rng_state.restype = C.c_uint64
    lib.dllm_sampler_get_rng_state.argtypes = [C.c_void_p]
    lib.dllm_sampler_set_rng_state.restype = None
    lib.dllm_sampler_set_rng_state.argtypes = [C.c_void_p, C.c_uint64]
    lib.sampler_create.restype = C.c_void_p
    lib.sampler_create.argtypes = [C.POINTER(SamplerConfig)]
    lib.sampler_free.restype = None
    lib.sampler_free.argtypes = [C.c_void_p]
    lib.sampler_sample.restype = C.c_int
    lib.sampler_sample.argtypes = [C.c_void_p, C.c_void_p, C.c_int]
    lib.greedy_sample.restype = C.c_int
    lib.greedy_sample.argtypes = [C.c_void_p, C.c_int]
    for name in ("sampler_apply_repetition_penalty", "sampler_apply_presence_penalty"):
        f = getattr(lib, name)
        f.restype = None
        f.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_float]
    _lib = lib
    return lib


def set_timing_events(before=None, after=None):
    """Has every later sampling call record the two torch.cuda.Event objects right before and
    right after the cluster kernel (None, None switches it off)."""
    b = None if before is None else before.cuda_event
    a = None if after is None else after.cuda_event
    rc = load_library().dllm_cuda_set_timing_events(b, a)
    if rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_set_timing_events: {STATUS_NAMES.get(rc, rc)}")


FAULT_NONE, FAULT_COPY_WAIT, FAULT_EXCHANGE_WAIT, FAULT_PRODUCT_WAIT = 0, 1, 2, 8


def inject_wait_timeout(site: int, polls: int = 1) -> None:
    """Test hook: later sampling launches make one bounded wait run out (FAULT_COPY_WAIT,
    FAULT_EXCHANGE_WAIT or, in the int8 product, FAULT_PRODUCT_WAIT) after `polls` polls; FAULT_NONE switches it off."""
    rc = load_library().dllm_cuda_debug_inject_wait_timeout(int(site), int(polls))
    if rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_debug_inject_wait_timeout: {STATUS_NAMES.get(rc, rc)}")


def fail_allocations(count: int) -> None:
    """Test hook: the library's next `count` device allocations fail as out of memory."""
    rc = load_library().dllm_cuda_debug_fail_allocations(int(count))
    if rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_debug_fail_allocations: {STATUS_NAMES.get(rc, rc)}")


def set_debug_counters(tensor_or_none):
    """Points the kernels' diagnostic counters at a zeroed CUDA int64 tensor of >= 32 entries
    (or switches them off with None)."""
    ptr = None if tensor_or_none is None else tensor_or_none.data_ptr()
    rc = load_library().dllm_cuda_set_debug_counters(ptr)
    if rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_set_debug_counters: {STATUS_NAMES.get(rc, rc)}")


def version() -> str:
    return load_library().dllm_cuda_version().decode()


def make_params(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0, repetition=1.0, presence=0.0,
                frequency=0.0) -> SamplerParams:
    return SamplerParams(float(temperature), float(top_p), float(min_p), int(top_k),
                         float(repetition), float(presence), float(frequency))


# ---------------------------------------------------------------------------------------------
# drop-in sampler (host pointers, like DiskLLM's sampler.h)

class Sampler:
    """DiskLLM's `sampler` object (src/sampler.c:56-95) served by the CUDA library."""

    def __init__(self, temperature=0.7, top_k=40, top_p=0.9, min_p=0.0, seed=0):
        self._lib = load_library()
        cfg = SamplerConfig(float(temperature), int(top_k), float(top_p), float(min_p), int(seed))
        self._h = self._lib.sampler_create(C.byref(cfg))
        if not self._h:
            raise DllmError("sampler_create returned NULL")

    def close(self):
        if self._h:
            self._lib.sampler_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def rng_state(self) -> int:
        return int(self._lib.dllm_sampler_get_rng_state(self._h))

    @rng_state.setter
    def rng_state(self, v: int):
        self._lib.dllm_sampler_set_rng_state(self._h, int(v))

    def sample(self, logits: np.ndarray) -> int:
        a = np.ascontiguousarray(logits, dtype=np.float32)
        return int(self._lib.sampler_sample(self._h, a.ctypes.data, a.shape[0]))


def greedy_sample(logits: np.ndarray) -> int:
    a = np.ascontiguousarray(logits, dtype=np.float32)
    return int(load_library().greedy_sample(a.ctypes.data, a.shape[0]))


def apply_repetition_penalty(logits: np.ndarray, seen, penalty: float) -> None:
    """In place on a float32 numpy row, like src/sampler.c:21-33."""
    assert logits.dtype == np.float32 and logits.flags.c_contiguous
    ids = np.ascontiguousarray(seen, dtype=np.int32)
    load_library().sampler_apply_repetition_penalty(logits.ctypes.data, logits.shape[0],
                                                    ids.ctypes.data, ids.shape[0], penalty)


def apply_presence_penalty(logits: np.ndarray, seen, presence: float) -> None:
    """In place on a float32 numpy row, like src/sampler.c:35-52."""
    assert logits.dtype == np.float32 and logits.flags.c_contiguous
    ids = np.ascontiguousarray(seen, dtype=np.int32)
    load_library().sampler_apply_presence_penalty(logits.ctypes.data, logits.shape[0],
                                                  ids.ctypes.data, ids.shape[0], presence)


# ---------------------------------------------------------------------------------------------
# batched device entry point (torch tensors are only containers for device memory here)

def fill_desc(logits, uniforms, params=None, *, mask=None, hist_ids=None, hist_off=None,
              hist_max=None, row_params=None, topk_max=0, flags=0, token=None, probs=None,
              pen_logits=None, status=None, topk_ids=None, workspace=None) -> tuple[BatchDesc, object]:
    """Builds a dllm_batch_desc from CUDA tensors; returns (desc, token tensor)."""
    import torch

    assert logits.is_cuda and logits.dim() == 2
    rows, vocab = logits.shape
    if logits.dtype == torch.float32:
        dt = DTYPE_F32
    elif logits.dtype == torch.bfloat16:
        dt = DTYPE_BF16
    else:
        raise TypeError(f"unsupported logits dtype {logits.dtype}")
    assert logits.stride(1) == 1
    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=logits.device)
    if params is None:
        params = make_params()
    elif isinstance(params, dict):
        params = make_params(**params)
    d = BatchDesc()
    d.rows, d.vocab, d.row_stride, d.dtype = rows, vocab, logits.stride(0), dt
    d.logits = logits.data_ptr()
    if mask is not None:
        assert mask.dtype in (torch.int32, torch.uint32) and mask.is_cuda
        d.mask, d.mask_stride = mask.data_ptr(), mask.stride(0)
    if hist_ids is not None:
        assert hist_ids.dtype == torch.int32 and hist_off.dtype == torch.int64
        d.hist_ids, d.hist_off = hist_ids.data_ptr(), hist_off.data_ptr()
        if hist_max is None:
            hist_max = int((hist_off[1:] - hist_off[:-1]).max().item()) if rows else 0
        d.hist_max = int(hist_max)
    assert uniforms.dtype == torch.float32 and uniforms.is_cuda
    d.uniforms = uniforms.data_ptr()
    d.params = params
    if row_params is not None:
        d.row_params = row_params.data_ptr()
        d.topk_max = int(topk_max)
    d.flags = int(flags)
    d.token = token.data_ptr()
    if probs is not None:
        d.probs, d.probs_stride = probs.data_ptr(), probs.stride(0)
    if pen_logits is not None:
        d.pen_logits, d.pen_stride = pen_logits.data_ptr(), pen_logits.stride(0)
    if status is not None:
        d.status = status.data_ptr()
    if topk_ids is not None:
        d.topk_ids, d.topk_stride = topk_ids.data_ptr(), topk_ids.stride(0)
    if workspace is not None:
        d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return d, token


def workspace_bytes(logits, uniforms, params=None, **kw) -> int:
    """dllm_cuda_workspace_bytes for the same arguments as sample_batch."""
    d, _ = fill_desc(logits, uniforms, params, **kw)
    return int(load_library().dllm_cuda_workspace_bytes(C.byref(d)))


def sample_batch(logits, uniforms, params=None, *, stream=None, check=True, **kw):
    """Calls dllm_cuda_sample_batch on CUDA tensors.  Returns the int32 token tensor."""
    import torch

    d, token = fill_desc(logits, uniforms, params, **kw)
    if stream is None:
        stream = torch.cuda.current_stream(logits.device).cuda_stream
    rc = load_library().dllm_cuda_sample_batch(C.byref(d), C.c_void_p(stream))
    if check and rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_sample_batch: {STATUS_NAMES.get(rc, rc)} "
                        f"({load_library().dllm_cuda_last_error().decode()})")
    return token


def sample_batch_static(logits, uniforms, params=None, *, stream=None, check=True, **kw):
    """Calls dllm_cuda_sample_batch_static: the same sampling with the library's fixed scratch
    array instead of any allocation.  Returns (token tensor, status code)."""
    import torch

    d, token = fill_desc(logits, uniforms, params, **kw)
    if stream is None:
        stream = torch.cuda.current_stream(logits.device).cuda_stream
    rc = load_library().dllm_cuda_sample_batch_static(C.byref(d), C.c_void_p(stream))
    if check and rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_sample_batch_static: {STATUS_NAMES.get(rc, rc)} "
                        f"({load_library().dllm_cuda_last_error().decode()})")
    return token, rc


def params_array(rows_params, device):
    """list of dicts -> device tensor laid out as dllm_sampler_params[rows]"""
    import torch

    arr = (SamplerParams * len(rows_params))(*[make_params(**p) for p in rows_params])
    raw = np.frombuffer(bytes(arr), dtype=np.uint8).copy()
    return torch.from_numpy(raw).to(device)


def shard_candidates(logits, vocab_offset, vocab_total, k, params=None, *, stream=None, check=True, out=None,
                     **kw):
    """Step 1 of vocabulary-sharded sampling on this GPU's columns: returns (values float32
    [rows][k], global ids int32 [rows][k]) of each row's k best entries after mask and penalties.
    `logits` holds columns [vocab_offset, vocab_offset + logits.shape[1]); `mask` (if given) the
    words of those columns; history ids are global.  `out` = (vals, ids): contiguous [rows][k]
    tensors to write into (views of one buffer, for a single all-gather)."""
    import torch

    rows = logits.shape[0]
    dummy_u = torch.empty(max(rows, 1), dtype=torch.float32, device=logits.device)
    d, _ = fill_desc(logits, dummy_u, params, **kw)
    if out is not None:
        vals, ids = out
        assert vals.is_contiguous() and ids.is_contiguous() and vals.shape == (rows, k) and ids.shape == (rows, k)
        assert vals.dtype == torch.float32 and ids.dtype == torch.int32
    else:
        vals = torch.empty(rows, k, dtype=torch.float32, device=logits.device)
        ids = torch.empty(rows, k, dtype=torch.int32, device=logits.device)
    s = stream if stream is not None else torch.cuda.current_stream(logits.device).cuda_stream
    rc = load_library().dllm_cuda_shard_candidates(C.byref(d), int(vocab_offset), int(vocab_total), int(k),
                                                   vals.data_ptr(), ids.data_ptr(), s)
    if check and rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_shard_candidates: {STATUS_NAMES.get(rc, rc)} ({load_library().dllm_cuda_last_error().decode()})")
    return vals, ids


def _check(rc, name):
    if rc != DLLM_OK:
        raise DllmError(f"{name}: {STATUS_NAMES.get(rc, rc)} ({load_library().dllm_cuda_last_error().decode()})")


def peer_exchange_create(rows, k, world):
    """This rank's peer exchange buffer: (device pointer, 64-byte IPC handle as bytes)."""
    buf = C.c_void_p()
    h = (C.c_ubyte * 64)()
    _check(load_library().dllm_cuda_peer_exchange_create(int(rows), int(k), int(world), C.byref(buf), h),
           "dllm_cuda_peer_exchange_create")
    return buf.value, bytes(h)


def peer_exchange_open(handle: bytes):
    """Maps another rank's exchange buffer on this GPU; returns its device pointer here."""
    h = (C.c_ubyte * 64).from_buffer_copy(handle)
    p = C.c_void_p()
    _check(load_library().dllm_cuda_peer_exchange_open(h, C.byref(p)), "dllm_cuda_peer_exchange_open")
    return p.value


def shard_candidates_peer(logits, vocab_offset, vocab_total, k, params, peers_dev, rank, world, epoch, *,
                          stream=None, **kw):
    """dllm_cuda_shard_candidates_peer: this GPU's candidates of step `epoch` into every rank's
    exchange buffer (peers_dev: int64 CUDA tensor [world] of the buffers as mapped here)."""
    import torch

    rows = logits.shape[0]
    dummy_u = torch.empty(max(rows, 1), dtype=torch.float32, device=logits.device)
    d, _ = fill_desc(logits, dummy_u, params, **kw)
    s = stream if stream is not None else torch.cuda.current_stream(logits.device).cuda_stream
    _check(load_library().dllm_cuda_shard_candidates_peer(C.byref(d), int(vocab_offset), int(vocab_total), int(k),
                                                          peers_dev.data_ptr(), int(rank), int(world), int(epoch), s),
           "dllm_cuda_shard_candidates_peer")


def shard_candidates_peer_desc(desc, vocab_offset, vocab_total, k, peers_dev, rank, world, epoch, stream):
    """dllm_cuda_shard_candidates_peer on a batch descriptor already built by fill_desc (its
    uniforms and token fields are not read); `stream` is a raw cudaStream_t value."""
    _check(load_library().dllm_cuda_shard_candidates_peer(C.byref(desc), int(vocab_offset), int(vocab_total), int(k),
                                                          peers_dev.data_ptr(), int(rank), int(world), int(epoch),
                                                          stream),
           "dllm_cuda_shard_candidates_peer")


def merge_sample_peer(rows, world, k, local_buf, epoch, uniforms, params, *, row_params=None, token=None,
                      status=None, stream=None):
    """dllm_cuda_merge_sample_peer over this rank's exchange buffer for step `epoch`."""
    import torch

    if isinstance(params, dict):
        params = make_params(**params)
    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=uniforms.device)
    s = stream if stream is not None else torch.cuda.current_stream(uniforms.device).cuda_stream
    rp = row_params.data_ptr() if row_params is not None else None
    st = status.data_ptr() if status is not None else None
    _check(load_library().dllm_cuda_merge_sample_peer(int(rows), int(world), int(k), local_buf, int(epoch),
                                                      C.byref(params), rp, uniforms.data_ptr(), token.data_ptr(), st, s),
           "dllm_cuda_merge_sample_peer")
    return token


def merge_sample(vals, ids, uniforms, params=None, *, row_params=None, token=None, status=None, stream=None,
                 check=True):
    """Step 3: tokens from all-gathered candidates vals / ids [nshards][rows][k].  `status` (int32
    [rows], optional) receives DLLM_ROW_ERR_TOPK_LARGE for per-row params the candidates cannot
    serve (temperature > 0 with top_k outside 1..k); those rows get the greedy token."""
    import torch

    nsh, rows, k = vals.shape
    assert vals.dtype == torch.float32 and ids.dtype == torch.int32 and vals.is_contiguous() and ids.is_contiguous()
    if params is None:
        params = make_params()
    elif isinstance(params, dict):
        params = make_params(**params)
    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=vals.device)
    s = stream if stream is not None else torch.cuda.current_stream(vals.device).cuda_stream
    rp = row_params.data_ptr() if row_params is not None else None
    st = status.data_ptr() if status is not None else None
    rc = load_library().dllm_cuda_merge_sample(rows, nsh, k, vals.data_ptr(), ids.data_ptr(), C.byref(params), rp,
                                               uniforms.data_ptr(), token.data_ptr(), st, s)
    if check and rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_merge_sample: {STATUS_NAMES.get(rc, rc)} ({load_library().dllm_cuda_last_error().decode()})")
    return token


# ---- grammar constraint (include/grammar.h) -------------------------------------------------

TOKEN_STR_CB = C.CFUNCTYPE(C.c_void_p, C.c_void_p, C.c_int)  # returns const char *


def _grammar_lib():
    lib = load_library()
    if not getattr(lib, "_grammar_typed", False):
        lib.diskllm_grammar_init_from_str.restype = C.c_void_p
        lib.diskllm_grammar_init_from_str.argtypes = [C.c_char_p]
        lib.diskllm_grammar_init_from_file.restype = C.c_void_p
        lib.diskllm_grammar_init_from_file.argtypes = [C.c_char_p]
        lib.diskllm_grammar_init_json.restype = C.c_void_p
        lib.diskllm_grammar_init_json.argtypes = []
        lib.diskllm_grammar_free.argtypes = [C.c_void_p]
        lib.diskllm_grammar_reset.argtypes = [C.c_void_p]
        lib.diskllm_grammar_accept_str.restype = C.c_bool
        lib.diskllm_grammar_accept_str.argtypes = [C.c_void_p, C.c_char_p]
        lib.diskllm_grammar_advance.argtypes = [C.c_void_p, C.c_char_p]
        lib.diskllm_grammar_is_finished.restype = C.c_bool
        lib.diskllm_grammar_is_finished.argtypes = [C.c_void_p]
        lib.diskllm_grammar_apply_mask.restype = C.c_int
        lib.diskllm_grammar_apply_mask.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, TOKEN_STR_CB, C.c_int]
        lib.dllm_grammar_build_bitmask.restype = C.c_int
        lib.dllm_grammar_build_bitmask.argtypes = [C.c_void_p, C.c_int, C.c_void_p, TOKEN_STR_CB, C.c_int, C.c_void_p]
        lib.dllm_grammar_vocab_create.restype = C.c_void_p
        lib.dllm_grammar_vocab_create.argtypes = [C.c_int, C.c_void_p, TOKEN_STR_CB, C.c_int]
        lib.dllm_grammar_vocab_free.argtypes = [C.c_void_p]
        lib.dllm_grammar_build_bitmask_cached.restype = C.c_int
        lib.dllm_grammar_build_bitmask_cached.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        lib._grammar_typed = True
    return lib


class Grammar:
    """DiskLLM's grammar constraint (diskllm_grammar_*) with the bitmask builder."""

    def __init__(self, text: str | None = None, *, json_mode: bool = False):
        lib = _grammar_lib()
        self._lib = lib
        self._g = lib.diskllm_grammar_init_json() if json_mode else lib.diskllm_grammar_init_from_str(
            text.encode() if text is not None else None)
        if not self._g:
            raise DllmError("diskllm_grammar_init failed")

    def __del__(self):
        if getattr(self, "_g", None):
            self._lib.diskllm_grammar_free(self._g)
            self._g = None

    def reset(self):
        self._lib.diskllm_grammar_reset(self._g)

    def accept(self, piece: bytes) -> bool:
        return bool(self._lib.diskllm_grammar_accept_str(self._g, piece))

    def advance(self, piece: bytes):
        self._lib.diskllm_grammar_advance(self._g, piece)

    def finished(self) -> bool:
        return bool(self._lib.diskllm_grammar_is_finished(self._g))

    def bitmask(self, pieces, eos: int) -> tuple[np.ndarray, int]:
        """(uint32 words, allowed count) for a vocabulary given as a list of bytes (None: no piece)."""
        cb, keep = _pieces_callback(pieces)
        words = np.zeros((len(pieces) + 31) // 32, dtype=np.uint32)
        n = self._lib.dllm_grammar_build_bitmask(self._g, len(pieces), None, cb, eos, words.ctypes.data)
        return words, n

    def apply_mask(self, logits: np.ndarray, pieces, eos: int) -> int:
        cb, keep = _pieces_callback(pieces)
        assert logits.dtype == np.float32 and logits.flags.c_contiguous
        return self._lib.diskllm_grammar_apply_mask(self._g, logits.ctypes.data, len(pieces), None, cb, eos)


class GrammarVocab:
    """Pieces read once (dllm_grammar_vocab_create) for per-step bitmasks without callbacks."""

    def __init__(self, pieces, eos: int):
        lib = _grammar_lib()
        self._lib = lib
        cb, keep = _pieces_callback(pieces)
        self.n = len(pieces)
        self._v = lib.dllm_grammar_vocab_create(len(pieces), None, cb, eos)
        if not self._v:
            raise DllmError("dllm_grammar_vocab_create failed")

    def __del__(self):
        if getattr(self, "_v", None):
            self._lib.dllm_grammar_vocab_free(self._v)
            self._v = None

    def bitmask(self, grammar: Grammar, out: np.ndarray | None = None) -> tuple[np.ndarray, int]:
        words = out if out is not None else np.zeros((self.n + 31) // 32, dtype=np.uint32)
        n = self._lib.dllm_grammar_build_bitmask_cached(grammar._g, self._v, words.ctypes.data)
        return words, n


def _pieces_callback(pieces):
    """A get_token_str callback over NUL-terminated copies of `pieces` (kept alive by the caller
    through the second return value)."""
    bufs = [None if p is None else C.create_string_buffer(p) for p in pieces]
    addrs = [None if b is None else C.addressof(b) for b in bufs]

    def get(_ctx, i):
        return addrs[i]

    return TOKEN_STR_CB(get), bufs


def lmhead_logits(h, w, *, norm_w=None, eps=1e-6, add_one=False, softcap=0.0, logits=None, stream=None, check=True):
    """Final RMSNorm + logits matvec + softcap (dllm_cuda_lmhead_logits): h fp32 [rows][hidden],
    w [vocab][hidden] fp32 / bf16 / fp16 (CUDA tensors); returns fp32 logits [rows][vocab]."""
    import torch

    rows, hidden = h.shape
    vocab = w.shape[0]
    assert h.dtype == torch.float32 and h.is_contiguous() and w.is_contiguous() and w.shape[1] == hidden
    wdt = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: 2}[w.dtype]
    if logits is None:
        logits = torch.empty(rows, vocab, dtype=torch.float32, device=h.device)
    s = stream if stream is not None else torch.cuda.current_stream(h.device).cuda_stream
    rc = load_library().dllm_cuda_lmhead_logits(rows, hidden, vocab, h.data_ptr(),
                                                None if norm_w is None else norm_w.data_ptr(), float(eps),
                                                int(bool(add_one)), w.data_ptr(), wdt, float(softcap),
                                                logits.data_ptr(), s)
    if check and rc != DLLM_OK:
        raise DllmError(f"dllm_cuda_lmhead_logits: {STATUS_NAMES.get(rc, rc)} "
                        f"({load_library().dllm_cuda_last_error().decode()})")
    return logits


# ---- int8 LM head -----------------------------------------------------------------------------
#
# These calls serve decode steps of a few microseconds, so their checks are written to cost little:
# messages are only formatted where a check fails, and devices are compared by index.

_FLOATS = None


def _float_code(dtype):
    """DTYPE_* of a torch dtype, None for others."""
    global _FLOATS
    if _FLOATS is None:
        import torch

        _FLOATS = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}
    return _FLOATS.get(dtype)


def _vector(t, n, dtype, dev, name):
    """Pointer of a contiguous vector of n elements on device `dev` (an index)."""
    if t.dtype is not dtype or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        raise DllmError(f"{name}: a contiguous {dtype} tensor of {n} elements on cuda:{dev} is needed")
    return t.data_ptr()


def _flags(t, n, dev, name):
    """Pointer of n contiguous bytes used as truth values."""
    import torch

    return _vector(t, n, torch.bool if t.dtype is torch.bool else torch.uint8, dev, name)


def _codes(t, dev, name):
    """(pointer, rows, cols, stride) of int8 rows that start on multiples of 16 bytes."""
    import torch

    if t.dtype is not torch.int8 or t.get_device() != dev or t.dim() != 2:
        raise DllmError(f"{name}: int8 rows on cuda:{dev} are needed")
    rows, cols = t.shape
    stride, inner = t.stride()
    if rows <= 1:  # the stride of a single row is not used
        stride = (cols + 15) // 16 * 16
    ptr = t.data_ptr()
    if (inner != 1 and cols > 1) or ptr % 16 or stride % 16 or stride < cols:
        raise DllmError(f"{name}: contiguous rows that start on multiples of 16 bytes are needed "
                        "(quantize_rows_i8 lays them out so)")
    return ptr, rows, cols, stride


def _scratch(ws, dev):
    """(pointer, bytes) of a workspace."""
    if ws.get_device() != dev or not ws.is_contiguous():
        raise DllmError(f"workspace: a contiguous tensor on cuda:{dev} is needed")
    return ws.data_ptr(), ws.numel() * ws.element_size()


_torch_c = None


def _torch_calls():
    """(current raw stream of a device, current device, device guard) of torch."""
    global _torch_c
    if _torch_c is None:
        import torch

        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # without making a Stream object
        _torch_c = (raw or (lambda i: torch.cuda.current_stream(i).cuda_stream), torch.cuda.current_device,
                    torch.cuda.device)
    return _torch_c


def _call(name, dev, *args):
    """Runs a library call on the current stream of device `dev`, with `dev` current."""
    raw_stream, current, guard = _torch_calls()
    f = getattr(load_library(), name)
    if current() == dev:
        rc = f(*args, raw_stream(dev))
    else:
        with guard(dev):
            rc = f(*args, raw_stream(dev))
    if rc != DLLM_OK:
        _check(rc, name)


def _on_stream(function):
    """`stream`: a raw cudaStream_t that the call runs on; what it allocates then belongs to that stream too
    (memory of the current one could be reused there while the call still works with it)."""
    @functools.wraps(function)
    def on_stream(*args, stream=None, **kw):
        if stream is None:
            return function(*args, **kw)
        import torch

        dev = next(t.device for t in (*args, *kw.values()) if isinstance(t, torch.Tensor))
        s = torch.cuda.ExternalStream(int(stream), dev) if int(stream) else torch.cuda.default_stream(dev)
        with torch.cuda.stream(s):
            return function(*args, **kw)
    return on_stream


_workspaces = threading.local()


def _workspace(nbytes, device, dev):
    """Scratch of a call on the current stream: this thread's buffer of the (device, stream), grown as
    needed; during a stream capture a tensor of its own, which the graph's pool keeps."""
    import torch

    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    held, key = _workspaces.__dict__, (dev, _torch_calls()[0](dev))
    ws = held.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = held[key] = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws


@_on_stream
def quantize_rows_i8(x, *, norm=False, norm_w=None, eps=1e-6, add_one=False, q=None, scale=None):
    """Rows to int8 codes with a scale each (dllm_cuda_quantize_rows_i8): x [rows][cols] fp32 / bf16 /
    fp16, RMS-normalised first when `norm`.  Returns (codes int8 [rows][cols], scale fp32 [rows]); the
    codes' rows start on multiples of 16 bytes."""
    import torch

    code, dev = _float_code(x.dtype), x.get_device()
    if dev < 0 or x.dim() != 2 or code is None:
        raise DllmError("x: a 2-D fp32, bf16 or fp16 CUDA tensor is needed")
    rows, cols = x.shape
    x_stride, inner = x.stride()
    if cols < 1 or (inner != 1 and cols > 1):
        raise DllmError("x: contiguous rows of at least one element are needed")
    if q is None:
        ld = (cols + 15) // 16 * 16
        q = x.new_empty((rows, ld), dtype=torch.int8)
        qp = q.data_ptr()
        if ld != cols:
            q = q[:, :cols]
    else:
        qp, qr, qc, ld = _codes(q, dev, "q")
        if (qr, qc) != (rows, cols):
            raise DllmError("q: the shape of x is needed")
    if scale is None:
        scale = x.new_empty(rows, dtype=torch.float32)
        sp = scale.data_ptr()
    else:
        sp = _vector(scale, rows, torch.float32, dev, "scale")
    _call("dllm_cuda_quantize_rows_i8", dev, rows, cols, x.data_ptr(), x_stride if rows > 1 else cols, code,
          bool(norm), None if norm_w is None else _vector(norm_w, cols, torch.float32, dev, "norm_w"), eps, bool(add_one),
          qp, ld, sp)
    return q, scale


@_on_stream
def matmul_i8(a, a_scale, b, b_scale, *, softcap=0.0, out=None, out_dtype=None, status=None):
    """out[i][j] = a_scale[i] b_scale[j] sum_k a[i][k] b[j][k] (dllm_cuda_matmul_i8): int8 codes a
    [m][k], b [n][k] as quantize_rows_i8 gives them, fp32 scales; out fp32 (default), bf16 or fp16."""
    import torch

    dev = a.get_device()
    if dev < 0:
        raise DllmError("a: a CUDA tensor is needed")
    ap, m, k, lda = _codes(a, dev, "a")
    bp, n, kb, ldb = _codes(b, dev, "b")
    if k != kb:
        raise DllmError(f"a has {k} columns, b {kb}")
    if out is None:
        out = a.new_empty((m, n), dtype=out_dtype or torch.float32)
        code, ldo = _float_code(out.dtype), n
    else:
        code = _float_code(out.dtype)
        if out.get_device() != dev or out.shape != (m, n) or (n > 1 and out.stride(1) != 1) or \
                (out_dtype is not None and out.dtype is not out_dtype):
            raise DllmError(f"out: contiguous rows [{m}][{n}] are needed")
        ldo = out.stride(0) if m > 1 else n
    if code is None:
        raise DllmError("out: fp32, bf16 or fp16 is needed")
    _call("dllm_cuda_matmul_i8", dev, m, n, k, ap, lda, _vector(a_scale, m, torch.float32, dev, "a_scale"), bp,
          ldb, _vector(b_scale, n, torch.float32, dev, "b_scale"), softcap, out.data_ptr(), ldo, code,
          None if status is None else _vector(status, 1, torch.int32, dev, "status"))
    return out


@_on_stream
def lmhead_logits_i8(h, w, w_scale, *, norm_w=None, eps=1e-6, add_one=False, softcap=0.0, logits=None, status=None,
                     workspace=None):
    """lmhead_logits with int8 output weights (dllm_cuda_lmhead_logits_i8): h fp32 [rows][hidden], w int8
    [vocab][hidden] and w_scale fp32 [vocab] from quantize_rows_i8; returns fp32 logits [rows][vocab]."""
    import torch

    dev = h.get_device()
    if dev < 0 or h.dim() != 2 or h.dtype is not torch.float32 or not h.is_contiguous():
        raise DllmError("h: a contiguous fp32 [rows][hidden] CUDA tensor is needed")
    rows, hidden = h.shape
    wp, vocab, hw, ldw = _codes(w, dev, "w")
    if hidden != hw:
        raise DllmError(f"h has {hidden} columns, w {hw}")
    if logits is None:
        logits = h.new_empty((rows, vocab))
    if workspace is None:
        workspace = _workspace(load_library().dllm_cuda_lmhead_i8_workspace_bytes(rows, hidden), h.device, dev)
    _call("dllm_cuda_lmhead_logits_i8", dev, rows, hidden, vocab, h.data_ptr(),
          None if norm_w is None else _vector(norm_w, hidden, torch.float32, dev, "norm_w"), eps, bool(add_one), wp, ldw,
          _vector(w_scale, vocab, torch.float32, dev, "w_scale"), softcap,
          _vector(logits, rows * vocab, torch.float32, dev, "logits"),
          None if status is None else _vector(status, 1, torch.int32, dev, "status"), *_scratch(workspace, dev))
    return logits


# ---- beam search ------------------------------------------------------------------------------

def fill_beam_desc(logits, scores, k, *, mask=None, finished=None, eos=-1, lengths=None, length_penalty=0.0, out=None,
                   out_finished=None, out_lengths=None, status=None, workspace=None):
    """Builds a dllm_beam_desc from CUDA tensors; returns (desc, (score, parent, token)).  The workspace is
    left out where none is given."""
    import torch

    code, dev = _float_code(logits.dtype), logits.get_device()
    if dev < 0 or logits.dim() != 2 or code is None:
        raise DllmError("logits: a 2-D fp32, bf16 or fp16 CUDA tensor is needed")
    if scores.dim() != 2:
        raise DllmError("scores: [batch][beams] is needed")
    batch, beams = scores.shape
    rows, vocab = logits.shape
    row_stride, inner = logits.stride()
    if rows != batch * beams:
        raise DllmError(f"logits have {rows} rows, scores {batch} x {beams}")
    if vocab > 1 and inner != 1:
        raise DllmError("logits: contiguous rows are needed")
    k = int(k)
    n = batch * k
    mask_ptr = mask_stride = 0
    if mask is not None:
        words = (vocab + 31) // 32
        if mask.dtype not in (torch.int32, torch.uint32) or mask.get_device() != dev or mask.dim() != 2 or \
                mask.shape[0] != rows or mask.shape[1] < words or (mask.shape[1] > 1 and mask.stride(1) != 1):
            raise DllmError(f"mask: int32 words [{rows}][{words}] on cuda:{dev} are needed")
        mask_ptr, mask_stride = mask.data_ptr(), mask.stride(0) if rows > 1 else words
    if out is None:
        buf = logits.new_empty((3, batch, max(k, 0)), dtype=torch.int32)
        score, parent, token = buf.unbind(0)
        out = (score.view(torch.float32), parent, token)
        p = buf.data_ptr()
        out_ptrs = (p, p + 4 * n, p + 8 * n)
    else:
        score, parent, token = out
        out_ptrs = (_vector(score, n, torch.float32, dev, "out score"), _vector(parent, n, torch.int32, dev, "out parent"),
                    _vector(token, n, torch.int32, dev, "out token"))
    d = BeamDesc(batch, beams, vocab, k, row_stride if rows > 1 else vocab, code, logits.data_ptr(), mask_ptr, mask_stride,
                 _vector(scores, rows, torch.float32, dev, "scores"),
                 None if finished is None else _flags(finished, rows, dev, "finished"), int(eos),
                 None if lengths is None else _vector(lengths, rows, torch.int32, dev, "lengths"), length_penalty,
                 *out_ptrs,
                 None if out_finished is None else _flags(out_finished, n, dev, "out_finished"),
                 None if out_lengths is None else _vector(out_lengths, n, torch.int32, dev, "out_lengths"),
                 None if status is None else _vector(status, rows, torch.int32, dev, "status"))
    if workspace is not None:
        d.workspace, d.workspace_bytes = _scratch(workspace, dev)
    return d, out


def beam_workspace_bytes(logits, scores, k, **kw) -> int:
    """dllm_cuda_beam_workspace_bytes for the same arguments as beam_select."""
    return int(load_library().dllm_cuda_beam_workspace_bytes(C.byref(fill_beam_desc(logits, scores, k, **kw)[0])))


@_on_stream
def beam_select(logits, scores, k, **kw):
    """The k best continuations of each sequence's beams (dllm_cuda_beam_select): logits [batch * beams]
    [vocab], scores fp32 [batch][beams].  Returns (score fp32, parent int32, token int32), each
    [batch][k], best rank first; a slot that nothing fills has (-inf, -1, -1).  Options: `mask`
    (packed allow-bits), `finished` and `eos` (ended beams), `lengths` and `length_penalty`, `out`
    (the three outputs), `out_finished`, `out_lengths`, `status`, `workspace`."""
    d, out = fill_beam_desc(logits, scores, k, **kw)
    dev, p = logits.get_device(), C.byref(d)
    if not d.workspace:
        ws = _workspace(load_library().dllm_cuda_beam_workspace_bytes(p), logits.device, dev)
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
    _call("dllm_cuda_beam_select", dev, p)
    return out


def _runs(t):
    """(row stride, segments, segment stride, run), strides and run in bytes, of a state [rows][...]
    whose inner dimensions are runs of one length at one stride."""
    esz = t.element_size()
    run, segs, seg_stride = esz, 1, 0
    strides = t.stride()
    for size, stride in zip(t.shape[:0:-1], strides[:0:-1]):
        if size == 1:
            continue
        if segs == 1 and stride * esz == run:
            run *= size
        elif segs == 1:
            segs, seg_stride = size, stride * esz
        elif stride * esz == segs * seg_stride:
            segs *= size
        else:
            raise DllmError("a state's rows have to be runs at one stride")
    return strides[0] * esz, segs, seg_stride, run


def _refuse_overlaps(groups, rows):
    """Raises where states of two groups share a byte (the library looks at those of one group)."""
    spans = sorted((p, p + (rows - 1) * row + (segs - 1) * seg + run, layout)
                   for layout, ptrs in groups.items() for row, segs, seg, run in (layout,) for p in ptrs)
    end, apart = 0, True
    for first, last, _ in spans:
        apart &= first >= end
        end = max(end, last)
    if apart:
        return
    for i, (a, a_end, la) in enumerate(spans):
        for b, _, lb in spans[i + 1:]:
            if b >= a_end:
                break
            if la != lb:  # one may lie in the other's gaps: run by run, in the order of their starts
                runs = [(p + np.add.outer(np.arange(rows) * row, np.arange(segs) * seg).ravel(), run)
                        for p, (row, segs, seg, run) in ((a, la), (b, lb))]
                start = np.concatenate([r[0] for r in runs])
                stop = np.concatenate([r[0] + r[1] for r in runs])
                order = np.argsort(start, kind="stable")
                if (stop[order][:-1] > start[order][1:]).any():
                    raise DllmError("states overlap")


@_on_stream
def beam_reorder(states, parents):
    """Moves states after their beams' parents, in place (dllm_cuda_beam_reorder): every tensor of
    `states` [batch * beams][...] gets row (s, b) from row (s, parents[s][b]); parents int32
    [batch][beams], -1 leaves the beam as it is.  A view, such as the used part of a cache, is moved
    without what lies around it.  States that share a byte are refused."""
    import torch

    dev = parents.get_device()
    if dev < 0 or parents.dim() != 2 or parents.dtype is not torch.int32 or not parents.is_contiguous():
        raise DllmError("parents: contiguous int32 [batch][beams] on the GPU is needed")
    batch, beams = parents.shape
    rows = batch * beams
    groups, seen = {}, set()
    for t in states:
        if t.get_device() != dev or t.dim() < 1 or t.shape[0] != rows:
            raise DllmError(f"a state of {rows} rows on cuda:{dev} is needed")
        if t.numel():
            ptr = t.data_ptr()
            if ptr in seen:
                raise DllmError("a state is given twice")
            seen.add(ptr)
            groups.setdefault(_runs(t), []).append(ptr)
    if len(groups) > 1:
        _refuse_overlaps(groups, rows)
    for (row, segs, seg, run), ptrs in groups.items():
        _call("dllm_cuda_beam_reorder", dev, batch, beams, parents.data_ptr(), len(ptrs),
              (C.c_void_p * len(ptrs))(*ptrs), row, segs, seg, run)
