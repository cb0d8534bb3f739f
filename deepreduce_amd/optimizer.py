"""Distributed optimizer / gradient-hook layer (GRACE DistributedOptimizer
equivalent — the part the reference leaves to grace_dl, SURVEY.md sect. 2.5).

Modes:
  * `reduce_gradients(model, grc)` — synchronous: call between backward and
    optimizer.step().
  * `DistributedOptimizer(opt, grc, model)` — wraps an optimizer; gradients
    are compressed+exchanged in .step() before the inner step.
  * hipGraph capture (MI355X-first): the leftmost-bloom/topk/qsgd pipeline
    is sync-free by construction (no .item()/.cpu() anywhere, payload sizes
    host-known), so the ENTIRE per-step exchange — compensate, top-k
    select, bloom insert/query, payload fusion, collective, fused
    multi-rank decompress, residual update — is captured once into a
    hipGraph and replayed as a single launch.  This removes the per-tensor
    launch storm (~10k dispatches/step measured eager on ResNet-50,
    profiles/) that dominates step time.  Enabled automatically when the
    pipeline is graph-safe; DEEPREDUCE_GRAPH=0 disables.

Gradients are compressed in float32 regardless of compute dtype (the wire
volume accounting and all codecs are float32, matching the reference).

params['clip_norm'] bounds the global gradient norm, by ops.clip_grad_norm_
(sync-free, so part of the captured graph).  params['clip_stage'] says where:
  * 'local' (default): each rank's own gradients, before they enter the
    residual memory, where an outlier would otherwise stay;
  * 'reduced': the exchanged gradients, which are the same on every rank.
The norm before clipping is left in `grc.last_grad_norm`, on the device, a
tensor of its own for each step.
"""
from __future__ import annotations

import os

import torch

from .ops import clip_grad_norm_
from .ops.language import TYPES

__all__ = ["reduce_gradients", "DistributedOptimizer"]


def reduce_gradients(model: torch.nn.Module, grc, names=None, fused: bool = True):
    """Compress+exchange every .grad in place.  Returns total wire bytes.

    `fused` (default) routes through the communicator's step_many — the
    whole-model bucket-fused exchange (one collective per step instead of
    one per tensor).  Set False for the reference-style per-tensor loop.
    """
    params = [(n, p) for n, p in reversed(list(model.named_parameters()))
              if p.grad is not None]
    clip, stage = clip_options(grc)
    if clip is not None and stage == "local" and params:
        # what reaches the exchange below: the gradient itself, or its copy in 32 bits
        grads = [p.grad.data.float() for _, p in params]
        grc.last_grad_norm = clip_grad_norm_(grads, clip)
    else:
        grads = None
    if fused and hasattr(grc, "step_many") and os.environ.get("DEEPREDUCE_FUSED", "1") == "1":
        named = [(n, g) for (n, _), g in zip(params, grads or
                                             [p.grad.data.float() for _, p in params])]
        reduced = grc.step_many(named)
        for (name, p), r in zip(params, reduced):
            p.grad.data.copy_(r.view_as(p.grad.data))
        total_bytes = getattr(grc, "last_wire_bytes", 0)
    else:
        total_bytes = 0
        # reverse order: last layers' grads are ready first after backward
        for i, (name, p) in enumerate(params):
            g32 = grads[i] if grads else p.grad.data.float()
            reduced = grc.step(g32, name)
            p.grad.data.copy_(reduced.view_as(p.grad.data))
            total_bytes += getattr(grc, "last_wire_bytes", 0)
    if clip is not None and stage == "reduced" and params:
        grc.last_grad_norm = clip_reduced([p.grad.data for _, p in params], clip)
    return total_bytes


def clip_options(grc):
    """(clip_norm or None, clip_stage) of a communicator's params."""
    params = getattr(grc, "params", None) or {}
    return params.get("clip_norm"), params.get("clip_stage", "local")


def clip_reduced(grads, bound: float):
    """clip_grad_norm_ of exchanged gradients of any type: the exchange is in 32
    bits, so those that hold more lose nothing on the way."""
    parts = [g if g.dtype in TYPES else g.float() for g in grads]
    norm = clip_grad_norm_(parts, bound)
    for g, part in zip(grads, parts):
        if part is not g:
            g.copy_(part)
    return norm


def _graph_safe(grc) -> bool:
    """True when the configured pipeline has no host syncs or data-dependent
    payload sizes: leftmost-policy bloom (sync-free query), qsgd, plain
    topk/randomk/none — NOT polyfit (segment count depends on num_pos),
    p0/conflict_sets/random policies, or threshold sparsification."""
    if os.environ.get("DEEPREDUCE_GRAPH", "1") == "0":
        return False
    # Collectives inside hipGraph capture (RCCL) cannot be qualified on the
    # single-GPU boxes we test on — multi-rank capture stays opt-in.
    import torch.distributed as dist

    if dist.is_available() and dist.is_initialized() and dist.get_world_size() > 1:
        if os.environ.get("DEEPREDUCE_GRAPH_DIST", "0") != "1":
            return False
    comp = getattr(grc, "compressor", None)
    params = getattr(comp, "params", None)
    from .compressors import RandomKCompressor, ThresholdCompressor

    if params is None:  # bare sparsifier
        return not isinstance(comp, (ThresholdCompressor, RandomKCompressor))
    # threshold: data-dependent payload sizes would replay with stale
    # shapes; randomk: the per-step CPU reseed would freeze at the
    # captured step — both eager only
    if isinstance(getattr(comp, "sparsifier", None),
                  (ThresholdCompressor, RandomKCompressor)):
        return False
    mode = params.get("deepreduce")
    if not mode:
        return True
    value = params.get("value", "polyfit")
    index = params.get("index", "bloom")
    policy = params.get("policy", "leftmost")
    if mode in ("index", "both") and (index != "bloom" or policy != "leftmost"):
        return False
    if mode in ("value", "both") and value not in ("qsgd",):
        # polyfit/polyseg run a radix sort, which proved unstable inside
        # hipGraph capture at ResNet-50 scale (gpurun_out/b10); their
        # batched pipeline is at dense-baseline speed eager anyway
        return False
    if params.get("micro-benchmark"):
        return False  # timing prints sync
    if params.get("log_stats"):
        return False  # host-side JSONL logger would freeze inside the graph
    return True


class DistributedOptimizer:
    """Optimizer wrapper: exchange compressed grads, then inner step.

    On ROCm, the exchange is hipGraph-captured after `graph_warmup` eager
    steps when the pipeline is graph-safe (see _graph_safe); capture
    failure falls back to eager permanently.
    """

    def __init__(self, optimizer: torch.optim.Optimizer, grc, model: torch.nn.Module,
                 use_graph: bool | None = None, graph_warmup: int = 3):
        self.optimizer = optimizer
        self.grc = grc
        self.model = model
        self.last_wire_bytes = 0
        self._graph = None
        self._graph_calls = 0
        self._graph_warmup = max(2, graph_warmup)  # residuals must exist
        self._use_graph = use_graph if use_graph is not None else _graph_safe(grc)
        self._graph_wire_bytes = 0
        self._graph_norm = None  # what the captured exchange writes its gradient norm to

    def zero_grad(self, set_to_none: bool = True):
        if not set_to_none:
            grads = [p.grad for p in self.model.parameters() if p.grad is not None]
            if grads:
                torch._foreach_zero_(grads)  # one fused launch, not one per tensor
                return
        self.optimizer.zero_grad(set_to_none=set_to_none)

    def _exchange(self):
        if not (self._use_graph and torch.cuda.is_available()
                and next(self.model.parameters()).is_cuda):
            self.last_wire_bytes = reduce_gradients(self.model, self.grc)
            return
        if self._graph is not None:
            if self._grad_ptrs() != self._graph_grad_ptrs:
                # gradient storages changed (e.g. zero_grad(set_to_none=True)
                # reallocated them): the captured pointers are stale —
                # invalidate and re-capture below.  If it keeps happening
                # (unstable grad storages every step), graphs can't help:
                # stay eager.
                self._graph = None
                self._recaptures = getattr(self, "_recaptures", 0) + 1
                if self._recaptures > 3:
                    self._use_graph = False
                    self.last_wire_bytes = reduce_gradients(self.model, self.grc)
                    return
            else:
                self._replay(self._graph)
                return
        self._graph_calls += 1
        if self._graph_calls <= self._graph_warmup:
            self.last_wire_bytes = reduce_gradients(self.model, self.grc)
            return
        # Capture.  Storage stability: p.grad buffers (zero_grad
        # set_to_none=False keeps them), residual buffers (ResidualMemory
        # updates in place), and graph-pool intermediates.  Canonical
        # recipe: warm the exact capture path up on a side stream first.
        # The warmup run mutates live state (p.grad <- reduced values,
        # residual updated), so snapshot grads + residuals before it and
        # restore before capturing: the captured pass then compresses the
        # pristine gradients exactly once, and the residual sees exactly
        # one update this step.
        try:
            grads, gsnap, rsnap = self._snapshot_state()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                reduce_gradients(self.model, self.grc)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            self._restore_state(grads, gsnap, rsnap)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._graph_wire_bytes = reduce_gradients(self.model, self.grc)
            self._graph_norm = self.last_grad_norm
            # capture RECORDS without executing: replay once so this step's
            # exchange actually happens (on the restored, pristine grads —
            # exactly one compress + one residual update this step)
            self._replay(g)
            self._graph = g
            self._graph_grad_ptrs = self._grad_ptrs()
        except Exception:
            self._use_graph = False
            self._graph = None
            torch.cuda.synchronize()
            self.last_wire_bytes = reduce_gradients(self.model, self.grc)

    def _replay(self, graph):
        graph.replay()
        self.last_wire_bytes = self._graph_wire_bytes
        if self._graph_norm is not None:
            # a tensor of this step's own: the next replay overwrites the graph's
            self.grc.last_grad_norm = self._graph_norm.clone()

    def _snapshot_state(self):
        """Clone p.grad buffers and residual-memory tensors (pre-warmup)."""
        grads = [p.grad for p in self.model.parameters() if p.grad is not None]
        gsnap = [g.detach().clone() for g in grads]
        mem = getattr(self.grc, "memory", None)
        rsnap = None
        if mem is not None and hasattr(mem, "residuals"):
            rsnap = {k: v.detach().clone() for k, v in mem.residuals.items()}
        return grads, gsnap, rsnap

    def _restore_state(self, grads, gsnap, rsnap):
        for g, s in zip(grads, gsnap):
            g.copy_(s)
        mem = getattr(self.grc, "memory", None)
        if rsnap is not None and mem is not None:
            for k, s in rsnap.items():
                r = mem.residuals.get(k)
                if r is not None and r.shape == s.shape:
                    r.copy_(s)
            # names whose residual buffers appeared during warmup (first
            # flat-pool build) started the warmup at zero: reset them
            for k, r in mem.residuals.items():
                if k not in rsnap:
                    r.zero_()
            for pool in getattr(mem, "_pools", {}).values():
                pool["c"] = None  # transient alias: never reuse post-restore

    def _grad_ptrs(self):
        return tuple(p.grad.data_ptr() for p in self.model.parameters()
                     if p.grad is not None)

    def step(self, closure=None):
        self._exchange()
        return self.optimizer.step(closure)

    @property
    def last_grad_norm(self):
        """The last step's gradient norm before clipping, a scalar on the
        device; None without params['clip_norm']."""
        return getattr(self.grc, "last_grad_norm", None)

    @property
    def param_groups(self):
        return self.optimizer.param_groups

    def state_dict(self):
        sd = {"optimizer": self.optimizer.state_dict()}
        mem = getattr(self.grc, "memory", None)
        if mem is not None:
            sd["memory"] = mem.state_dict()
        return sd

    def load_state_dict(self, sd):
        self.optimizer.load_state_dict(sd["optimizer"])
        mem = getattr(self.grc, "memory", None)
        if mem is not None and "memory" in sd:
            mem.load_state_dict(sd["memory"])
        self._graph = None  # residual storages changed: re-capture
