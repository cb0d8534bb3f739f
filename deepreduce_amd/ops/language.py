"""Language-model operators: attention over packed documents, rotary
positions, the global gradient norm and clipping.

Like the rest of `ops`: HIP kernels (ops/src/attention.hip, rotary.hip,
grad_norm.hip) on a GPU, the torch reference on the CPU.  Everything runs on
the current stream without a host synchronisation and can be captured into a
hipGraph; wrong arguments raise ValueError.  A backward pass is captured while
no eager graph of the same leaves is alive: with one, torch ends the process,
which attention and rotary refuse where the leaves are their own inputs.
Attention and rotary have no forward-mode derivatives and refuse dual tensors;
on a GPU none of the operators can be traced (torch.jit.trace, make_fx), since
a trace holds torch operations only.
"""
from __future__ import annotations

import bisect
import math

import torch

from . import reference as _ref

TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _hip(t):
    """The extension if `t` is on a GPU, None on the CPU."""
    from deepreduce_amd import ops

    return ops._hip if ops._want_hip(t) else None


def _check(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

class _Attention(torch.autograd.Function):
    """The CPU path; the extension has its own."""

    @staticmethod
    def forward(ctx, q, k, v, documents, slopes, causal, scale):
        out, lse = _ref.attention_forward(q, k, v, documents, slopes, causal, scale)
        ctx.save_for_backward(q, k, v, lse, documents, slopes)
        ctx.options = (causal, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        grads = _ref.attention_backward(dout, *ctx.saved_tensors, *ctx.options)
        return (*grads, None, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              documents: torch.Tensor | None = None, slopes: torch.Tensor | None = None,
              causal: bool = False, scale: float | None = None) -> torch.Tensor:
    """Softmax attention over packed documents, with a distance bias.

    q [B, Sq, Hq, D]; k, v [B, Sk, Hkv, D] with Sq <= Sk, Hkv dividing Hq and
    D a multiple of 8 up to 128; float32, bfloat16 or float16, any strides
    (heads that do not start at 16-byte addresses are copied first).  The
    queries are the last Sq of the Sk positions.  Returns [B, Sq, Hq, D];
    differentiable in q, k and v.

    documents: int32 [B, Sk], the document of each position in any order; a
        query sees its own document's keys, and nobody sees a negative one
        (padding).  A query that sees no key gives 0 and zero gradients, and
        nothing behind the mask, infinities and NaN included, reaches a result.
    slopes: float32 [Hq], constants; head h's scores get
        -slopes[h] * |query position - key position|.
    causal: a query sees no later position.
    scale: factor of the scores, D ** -0.5 by default.

    On a GPU scores, sums and statistics have 32 bits.  For 16-bit inputs the
    probabilities, and in the backward pass their gradients, are rounded to the
    inputs' type once more before their products, as the matrix cores take
    them: results are off by about 1.4 times their own rounding.
    """
    hip = _hip(q)
    if hip:
        return hip.attention(q, k, v, documents, slopes, causal, scale)
    _check(all(t.dim() == 4 for t in (q, k, v)),
           "attention: q, k and v must be [batch, length, heads, head size]")
    _check(q.dtype in TYPES, f"attention: q must be float32, bfloat16 or float16, got {q.dtype}")
    _check(k.dtype == q.dtype and v.dtype == q.dtype,
           f"attention: q, k and v have types {q.dtype}, {k.dtype}, {v.dtype}")
    _check(k.device == q.device and v.device == q.device,
           "attention: q, k and v are on different devices")
    b, sq, hq, d = q.shape
    _check(k.shape == v.shape and k.shape[0] == b and k.shape[3] == d,
           f"attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    sk, hkv = k.shape[1:3]
    _check(d % 8 == 0 and 8 <= d <= 128,
           f"attention: the head size must be a multiple of 8 from 8 to 128, got {d}")
    _check(hkv >= 1 and hq % hkv == 0,
           f"attention: {hkv} key-value heads do not divide {hq} query heads")
    _check(sq <= sk, f"attention: {sq} queries over {sk} keys; queries are the last positions")
    _check(sk < 1 << 30, "attention: too many keys")
    if documents is not None:
        _check(documents.dtype == torch.int32 and documents.shape == (b, sk)
               and documents.device == q.device,
               f"attention: documents must be int32 [{b}, {sk}] on q's device")
    if slopes is not None:
        _check(slopes.dtype == torch.float32 and slopes.shape == (hq,)
               and slopes.device == q.device,
               f"attention: slopes must be float32 [{hq}] on q's device")
        _check(not slopes.requires_grad, "attention: slopes are constants and get no gradient")
    scale = d ** -0.5 if scale is None else float(scale)
    _check(math.isfinite(scale), "attention: scale must be finite")
    return _Attention.apply(q, k, v, documents, slopes, bool(causal), scale)


# --------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------

def rotary_frequencies(dim: int, base: float = 10000.0, factor: float = 1.0,
                       trained_length: int | None = None, low: float = 1.0, high: float = 32.0,
                       device=None) -> torch.Tensor:
    """The float64 [dim / 2] angles that one position turns each pair by.

    base ** (-2 i / dim), scaled for contexts `factor` times as long as those
    trained on: all divided by `factor`, or, where `trained_length` is given,
    by parts: pairs that turn more than `high` times within it keep their
    frequency, pairs that turn less than `low` times are divided by `factor`,
    and those between get a linear mixture of the two.
    """
    _check(dim >= 2 and dim % 2 == 0, f"rotary_frequencies: dim must be even, got {dim}")
    _check(base > 1 and factor >= 1 and high > low >= 0,
           "rotary_frequencies: needs base > 1, factor >= 1 and high > low >= 0")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    f = float(base) ** (-i / dim)
    if trained_length is None:
        f = f / factor
    else:
        _check(trained_length >= 1, "rotary_frequencies: trained_length must be positive")
        turns = trained_length * f / (2 * math.pi)
        kept = ((turns - low) / (high - low)).clamp(0, 1)
        f = f * (kept + (1 - kept) / factor)
    return f.to(device)


class _Rotary(torch.autograd.Function):
    """The CPU path; the extension has its own."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved):
        ctx.save_for_backward(positions, frequencies)
        ctx.interleaved = interleaved
        return tuple(_ref.rotary([q, k], positions, frequencies, interleaved, False))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        grads = _ref.rotary([dq, dk], *ctx.saved_tensors, ctx.interleaved, True)
        return (*grads, None, None, None)


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
           frequencies: torch.Tensor, interleaved: bool = False):
    """(q, k) with the heads' first 2 * len(frequencies) values turned by position.

    q, k [B, S, heads, D] (any strides; other heads, same type): float32,
    bfloat16 or float16.  positions int32 or int64, [S] or [B, S], so they can
    restart with each document of a packed row.  frequencies float64
    (`rotary_frequencies`).  Pairs are values (i, i + n) of n frequencies, or
    (2 i, 2 i + 1) if interleaved.  Angles are formed in 64 bits, so far
    positions keep theirs.  Differentiable in q and k.
    """
    hip = _hip(q)
    if hip:
        return tuple(hip.rotary(q, k, positions, frequencies, interleaved))
    _check(q.dim() == 4 and k.dim() == 4 and q.shape[:2] == k.shape[:2]
           and q.shape[3] == k.shape[3],
           f"rotary: q {tuple(q.shape)} and k {tuple(k.shape)} must be "
           "[batch, length, heads, head size] with one batch, length and head size")
    _check(q.dtype in TYPES and k.dtype == q.dtype,
           f"rotary: q and k must be float32, bfloat16 or float16, got {q.dtype}, {k.dtype}")
    _check(len({t.device for t in (q, k, positions, frequencies)}) == 1,
           "rotary: q, k, positions and frequencies must be on one device")
    b, s, _, d = q.shape
    _check(positions.dtype in (torch.int32, torch.int64)
           and positions.shape in ((s,), (b, s)),
           f"rotary: positions must be int32 or int64, [{s}] or [{b}, {s}]")
    _check(frequencies.dtype == torch.float64 and frequencies.dim() == 1
           and 1 <= frequencies.numel() <= d // 2,
           f"rotary: frequencies must be float64 with 1 to {d // 2} values")
    _check(not frequencies.requires_grad, "rotary: frequencies are constants and get no gradient")
    _check(d % 2 == 0 and d <= 1024,
           f"rotary: the head size must be even and at most 1024, got {d}")
    return _Rotary.apply(q, k, positions.expand(b, s), frequencies, bool(interleaved))


# --------------------------------------------------------------------------
# the global gradient norm, and clipping
# --------------------------------------------------------------------------

def _list(tensors) -> list[torch.Tensor]:
    grads = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    _check(len(grads) > 0, "no tensors")
    return grads


def _check_gradients(grads, name: str) -> None:
    for t in grads:
        if t.dtype not in TYPES or t.layout != torch.strided or t.device != grads[0].device:
            raise ValueError(f"{name}: takes dense float32, bfloat16 or float16 tensors of one "
                             f"device, got {t.layout} {t.dtype} on {t.device}")


def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm of all values of all tensors: a float32 scalar on their device.

    Tensors of any shape, order and mixture of float32, bfloat16 and float16.
    Squares are added in 64 bits, in a fixed order.  A constant for both
    modes of differentiation.
    """
    grads = _list(tensors)
    hip = _hip(grads[0])
    if hip:
        return hip.grad_norm(grads)
    _check_gradients(grads, "grad_norm")
    return _ref.grad_norm([t.detach() for t in grads])


def clip_grad_norm(tensors, max_norm: float, out=None, dtype: torch.dtype | None = None):
    """(clipped, norm): the tensors times min(1, max_norm / norm), and their `grad_norm`.

    Writes to `out` (one tensor for each, of its shape and any of the three
    types; it may be the tensor itself, but the stretches of memory that
    outputs lie in, gaps included, may not overlap otherwise) or to new tensors
    of `dtype` (each one's own by default).  A norm that is infinite or NaN
    enters the product as it is: the one makes finite values 0 and infinities
    NaN, the other makes every value NaN.  Constants for both
    modes of differentiation.
    """
    grads, outs = _list(tensors), None if out is None else _list(out)
    max_norm = float(max_norm)
    _check(dtype is None or dtype in TYPES,
           f"clip_grad_norm: dtype must be float32, bfloat16 or float16, got {dtype}")
    hip = _hip(grads[0])
    if hip:
        new, norm = hip.clip_grad_norm(grads, max_norm, outs, dtype)
        return new if outs is None else outs, norm
    _check_gradients(grads, "clip_grad_norm")
    _check(max_norm >= 0, f"clip_grad_norm: max_norm must be 0 or more, got {max_norm}")
    _check(dtype is None or out is None, "clip_grad_norm: dtype is for new tensors, without out")
    if outs is None:
        outs = [torch.empty_like(t, dtype=dtype, requires_grad=False) for t in grads]
    _check_gradients(outs, "clip_grad_norm")
    _check(len(outs) == len(grads) and all(o.shape == t.shape for o, t in zip(outs, grads))
           and outs[0].device == grads[0].device,
           "clip_grad_norm: out must hold a tensor of each one's shape and device")
    _check_apart(grads, outs)
    norm = _ref.clip_grad_norm([t.detach() for t in grads], [t.detach() for t in outs], max_norm)
    if out is not None:
        torch.autograd.graph.increment_version(outs)
    return outs, norm


def clip_grad_norm_(tensors, max_norm: float) -> torch.Tensor:
    """`clip_grad_norm` in place; returns the norm that the tensors had."""
    grads = _list(tensors)
    return clip_grad_norm(grads, max_norm, out=grads)[1]


def _check_apart(grads, outs):
    """What is written may be read only as the same values' own input."""
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    for i, o in enumerate(outs):
        _check(all(n < 2 or s for n, s in zip(o.shape, o.stride())),
               f"clip_grad_norm: output {i} is expanded")
    written = sorted((*span(o), i) for i, o in enumerate(outs) if o.numel())
    for (_, end, i), (at, _, j) in zip(written, written[1:]):
        _check(at >= end, f"clip_grad_norm: outputs {i} and {j} share memory")
    ends = [end for _, end, _ in written]
    for j, t in enumerate(grads):
        if t.numel() == 0:
            continue
        at, end = span(t)
        n = bisect.bisect_right(ends, at)
        if n < len(written) and written[n][0] < end:
            o = outs[j]
            _check(written[n] == (at, end, j) and t.stride() == o.stride()
                   and t.dtype == o.dtype,
                   f"clip_grad_norm: gradient {j} shares memory with output {written[n][2]}")
