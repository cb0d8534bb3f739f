"""Language-model operators where their callers leave the common path: other
modes of differentiation and tracing, extreme and not finite values, rows of
zeros, block shapes of large inputs.  Oracles and tolerances are those of
test_language_ops.py where nothing else is said."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from deepreduce_amd import ops
from test_language_ops import (BOTH, E, TYPES, assert_within, attention_inputs, attention_oracle,
                               check_attention, half_step, pack)


# --------------------------------------------------------------------------
# what torch has to see
# --------------------------------------------------------------------------

def small_calls(device):
    """{name: (a call, its inputs)} of each operator."""
    q, k, v, _ = attention_inputs(1, 5, 7, 2, 1, 16, torch.float32, device)
    positions, frequencies = torch.arange(5, device=device), ops.rotary_frequencies(
        16, device=device)
    return {
        "attention": (lambda q, k, v, s: ops.attention(q, k, v, slopes=s),
                      (q, k, v, torch.tensor([0.5, 0.25], device=device))),
        "rotary": (lambda q, k, f: ops.rotary(q, k, positions, f)[0],
                   (q, k[:, :5], frequencies)),
        "grad_norm": (lambda a, b: ops.grad_norm([a, b]), (q, k)),
        "clip_grad_norm": (lambda a, b: ops.clip_grad_norm([a, b], 0.5)[0][1], (q, k)),
    }


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("name", ["attention", "rotary"])
def test_forward_derivatives_are_refused(device, name):
    """A result without a tangent would stand for a derivative of zero."""
    call, inputs = small_calls(device)[name]
    want = call(*inputs)
    with forward_ad.dual_level():
        for n, x in enumerate(inputs):
            duals = list(inputs)
            duals[n] = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError):
                call(*duals)
    assert torch.equal(call(*inputs), want)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("name", ["grad_norm", "clip_grad_norm"])
def test_norm_is_a_constant(device, name):
    call, inputs = small_calls(device)[name]
    with forward_ad.dual_level():
        duals = [forward_ad.make_dual(x, torch.ones_like(x)) for x in inputs]
        assert forward_ad.unpack_dual(call(*duals)).tangent is None
    assert not call(*[x.clone().requires_grad_(True) for x in inputs]).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["attention", "rotary", "grad_norm", "clip_grad_norm"])
def test_tracing_is_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    call, inputs = small_calls("cuda")[name]
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, inputs)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call)(*inputs)
    call(*inputs)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_tracing_on_the_cpu():
    for call, inputs in small_calls("cpu").values():
        traced = torch.jit.trace(call, inputs)
        other = tuple(x * 0.5 for x in inputs)
        assert torch.equal(traced(*other), call(*other))
