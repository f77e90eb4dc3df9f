"""Device-side decode loop for one sequence: the step sequence of DiskLLM's
diskllm_sample_grammar (src/core/sampler_api.c:48-73) -- mask, presence, repetition, sample --
followed by appending the sampled id to the history the next step penalises, all on the GPU.
The whole run of steps is captured once as a CUDA graph and replayed, so a step costs the
kernels' time and no host round trip.

The logits of step i are row i % R of a device ring (a real model writes them in place each step;
here they are given), the uniform of step i is uniforms[i] (one U[0,1) per step).

BeamLoop is the same for beam search: LM head with int8 weights, selection over beams and
vocabulary, states moved after their parents.
"""
from __future__ import annotations

import torch

from . import capi


class DecodeLoop:
    def __init__(self, logits_ring: torch.Tensor, uniforms: torch.Tensor, params: dict,
                 history: torch.Tensor, cap: int | None = None, mask_ring: torch.Tensor | None = None):
        assert logits_ring.is_cuda and logits_ring.dim() == 2
        self.dev = logits_ring.device
        self.ring = logits_ring
        self.mask_ring = mask_ring
        self.u = uniforms
        self.steps = uniforms.numel()
        self.params = params
        self.init_hist = history.to(self.dev, torch.int32).contiguous()
        self.cap = int(cap if cap is not None else self.init_hist.numel() + self.steps)
        assert self.cap >= self.init_hist.numel()
        self.hist_ids = torch.zeros(self.cap, dtype=torch.int32, device=self.dev)
        self.hist_off = torch.zeros(2, dtype=torch.int64, device=self.dev)
        self.init_off = torch.tensor([0, self.init_hist.numel()], dtype=torch.int64, device=self.dev)
        self.tokens = torch.empty(self.steps, dtype=torch.int32, device=self.dev)
        # scratch given to every call, so that nothing is allocated inside a capture
        nb = capi.workspace_bytes(self.ring[:1], self.u[:1], params, hist_ids=self.hist_ids, hist_off=self.hist_off,
                                  hist_max=self.cap)
        self.ws = torch.empty(max(nb, 256), dtype=torch.uint8, device=self.dev)
        self.graph = None

    def _reset(self):
        self.hist_ids[: self.init_hist.numel()].copy_(self.init_hist)
        self.hist_off.copy_(self.init_off)

    def _step(self, i: int):
        r = i % self.ring.shape[0]
        kw = {}
        if self.mask_ring is not None:
            kw["mask"] = self.mask_ring[r:r + 1]
        capi.sample_batch(self.ring[r:r + 1], self.u[i:i + 1], self.params, hist_ids=self.hist_ids,
                          hist_off=self.hist_off, hist_max=self.cap, token=self.tokens[i:i + 1],
                          workspace=self.ws, **kw)
        rc = capi.load_library().dllm_cuda_append_history(
            self.tokens[i:i + 1].data_ptr(), self.hist_ids.data_ptr(), self.hist_off.data_ptr(), self.cap,
            torch.cuda.current_stream(self.dev).cuda_stream)
        if rc != capi.DLLM_OK:
            raise capi.DllmError(f"dllm_cuda_append_history: {capi.STATUS_NAMES.get(rc, rc)}")

    def run_eager(self) -> torch.Tensor:
        """Every step launched from the host."""
        self._reset()
        for i in range(self.steps):
            self._step(i)
        return self.tokens

    def capture(self):
        """Records reset + all steps as one CUDA graph (after one eager step, which fixes the
        launch configuration outside the capture)."""
        self._reset()
        self._step(0)
        torch.cuda.synchronize(self.dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self._reset()
            for i in range(self.steps):
                self._step(i)
        return self

    def replay(self) -> torch.Tensor:
        if self.graph is None:
            self.capture()
        self.graph.replay()
        return self.tokens


class BeamLoop:
    """Beam search over `batch` sequences of `beams` beams.  A step takes the hidden states of every
    beam (entry i % R of hidden_ring [R][batch * beams][hidden], fp32), forms their logits with int8
    output weights (wq, w_scale from capi.quantize_rows_i8), selects the best `beams` continuations
    of each sequence, moves `states` (tensors [batch * beams][...], such as caches) and the token
    histories after their parents, and appends the new tokens.  The first step starts from one live
    beam per sequence.  A beam that has produced `eos` stays as it is.

    After a run: tokens [batch][beams][steps] int32 (best beam first; after an end the token is eos,
    in slots that nothing filled -1), scores [batch][beams], lengths and finished; and status
    [batch][beams] int32, DLLM_ROW_ERR_* bits of all steps: NONFINITE for a beam whose logits or score
    were not finite, so that it offered nothing (its place in the sequence's later steps may be
    another's), TIMEOUT for every beam where a wait of the LM head ran out.  Then the logits of a step
    are not meaningful, and tokens are -1 and scores NaN.  A run returns before the GPU is done; check()
    waits for it and raises where a status is not 0."""

    def __init__(self, hidden_ring: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, batch: int, beams: int,
                 steps: int, *, eos: int, length_penalty: float = 0.0, norm_w: torch.Tensor | None = None,
                 eps: float = 1e-6, add_one: bool = False, softcap: float = 0.0, states=(),
                 mask_ring: torch.Tensor | None = None):
        assert hidden_ring.is_cuda and hidden_ring.dim() == 3 and hidden_ring.shape[1] == batch * beams
        self.dev = hidden_ring.device
        self.ring, self.wq, self.w_scale = hidden_ring, wq, w_scale
        self.batch, self.beams, self.steps = batch, beams, steps
        self.eos, self.length_penalty = eos, length_penalty
        self.head = dict(norm_w=norm_w, eps=eps, add_one=add_one, softcap=softcap)
        self.states = list(states)
        self.mask_ring = mask_ring
        rows = batch * beams

        def buf(*shape, dtype=torch.int32):
            return torch.zeros(*shape, dtype=dtype, device=self.dev)

        self.scores, self.lengths = buf(batch, beams, dtype=torch.float32), buf(batch, beams)
        self.finished = buf(batch, beams, dtype=torch.uint8)
        self.parents, self.new = buf(batch, beams), buf(batch, beams)
        self.hist = buf(rows, steps)
        self.head_status, self.step_status = buf(1), buf(steps, batch, beams)
        self.first = torch.full((batch, beams), float("-inf"), device=self.dev)
        self.first[:, 0] = 0.0
        # buffers given to every call, so that nothing is allocated inside a capture
        self.logits = buf(rows, wq.shape[0], dtype=torch.float32)
        self.head_ws = buf(max(1, capi.load_library().dllm_cuda_lmhead_i8_workspace_bytes(rows, wq.shape[1])),
                           dtype=torch.uint8)
        self.beam_ws = buf(capi.beam_workspace_bytes(self.logits, self.scores, beams), dtype=torch.uint8)
        if mask_ring is not None:  # rows with a mask are dealt out differently
            masked = capi.beam_workspace_bytes(self.logits, self.scores, beams, mask=mask_ring[0])
            self.beam_ws = buf(max(masked, self.beam_ws.numel()), dtype=torch.uint8)
        self.graph = None

    @property
    def tokens(self) -> torch.Tensor:
        return self.hist.view(self.batch, self.beams, self.steps)

    @property
    def status(self) -> torch.Tensor:
        return (self.step_status & capi.ROW_ERR_NONFINITE).sum(0).clamp_(max=capi.ROW_ERR_NONFINITE).int() | self.head_status

    def check(self) -> torch.Tensor:
        """Waits for the run and raises DllmError where a step of it failed; the tokens."""
        status = self.status.cpu()
        if (status & capi.ROW_ERR_TIMEOUT).any():
            raise capi.DllmError("BeamLoop: a wait of the LM head ran out, the tokens are not valid")
        if status.any():
            raise capi.DllmError("BeamLoop: logits or scores that are not finite, in the sequences "
                                 f"{status.any(1).nonzero().view(-1).tolist()}")
        return self.tokens

    def _reset(self):
        self.scores.copy_(self.first)
        self.lengths.zero_()
        self.finished.zero_()
        self.head_status.zero_()
        self.step_status.zero_()

    def _end(self):
        """Where the LM head gave up nothing that looks like a result is left."""
        late = self.head_status != 0
        self.hist.masked_fill_(late, -1)
        self.scores.masked_fill_(late, float("nan"))

    def _step(self, i: int):
        r = i % self.ring.shape[0]
        capi.lmhead_logits_i8(self.ring[r], self.wq, self.w_scale, logits=self.logits, workspace=self.head_ws,
                              status=self.head_status, **self.head)
        capi.beam_select(self.logits, self.scores, self.beams, finished=self.finished, eos=self.eos,
                         mask=None if self.mask_ring is None else self.mask_ring[r],
                         lengths=self.lengths, length_penalty=self.length_penalty,
                         out=(self.scores, self.parents, self.new), out_finished=self.finished,
                         out_lengths=self.lengths, status=self.step_status[i], workspace=self.beam_ws)
        capi.beam_reorder([self.hist[:, :i], *self.states], self.parents)
        self.hist[:, i].copy_(self.new.view(-1))

    def run_eager(self) -> torch.Tensor:
        """Every step launched from the host."""
        self._reset()
        for i in range(self.steps):
            self._step(i)
        self._end()
        return self.tokens

    def capture(self):
        """Records reset + all steps as one CUDA graph.  Nothing runs on the states before it: the
        library is warmed up by one product and one selection on this loop's own buffers."""
        capi.lmhead_logits_i8(self.ring[0], self.wq, self.w_scale, logits=self.logits, workspace=self.head_ws, **self.head)
        self._reset()
        capi.beam_select(self.logits, self.scores, self.beams, out=(self.scores, self.parents, self.new),
                         workspace=self.beam_ws)
        torch.cuda.synchronize(self.dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self._reset()
            for i in range(self.steps):
                self._step(i)
            self._end()
        return self

    def replay(self) -> torch.Tensor:
        if self.graph is None:
            self.capture()
        self.graph.replay()
        return self.tokens
