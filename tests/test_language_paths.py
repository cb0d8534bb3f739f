"""The language-model operators in the framework's own paths, where a program
leaves the usual order of steps: evaluation before training, parameters of
other types, steps without gradients, more than one rank."""
import copy
import math

import pytest
import torch

import deepreduce_amd as dr
from deepreduce_amd import ops
from test_language_training import BOTH, POSITIONS, global_norm, make_grc, tiny_bert


# --------------------------------------------------------------------------
# BERT
# --------------------------------------------------------------------------

def bert_gradients(model, ids):
    model.zero_grad()
    out = model(ids)
    out.float().square().sum().backward()
    return [out.detach(), *[p.grad.clone() for p in model.parameters()]]


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("positions", POSITIONS)
def test_bert_trains_after_an_evaluation(device, positions):
    """Constants that the first call makes serve every later one."""
    ids = torch.randint(0, 97, (2, 20), generator=torch.Generator().manual_seed(0)).to(device)
    want = bert_gradients(tiny_bert(positions, device), ids)
    for moved in (False, True):
        model = tiny_bert(positions, device)
        if moved:  # a model whose parameters came to the device by themselves
            model._constants.clear()
        with torch.inference_mode():
            out = model(ids)
        for a, c in zip(bert_gradients(model, ids), want):
            assert torch.equal(a, c)
        assert torch.equal(out, want[0])
        for a, c in zip(bert_gradients(copy.deepcopy(model), ids), want):
            assert torch.equal(a, c)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("positions", ["rotary", "distance"])
def test_bert_constants(device, positions):
    """They are there before the first call, keep their type in a model of
    fewer bits and are not part of its state."""
    model = tiny_bert(positions, "cpu").to(device)
    at = model.tok.weight.device
    before = model._constants[at]
    assert before.dtype == (torch.float64 if positions == "rotary" else torch.float32)
    model = model.bfloat16()
    assert torch.equal(model._constants[at], before) and model._constants[at].dtype == before.dtype
    assert model(torch.zeros(1, 5, dtype=torch.int64, device=device)).dtype == torch.bfloat16
    names = {n for n, _ in model.named_parameters()} | {"head.weight"}
    assert set(model.state_dict()) == names
    with torch.device("meta"):
        empty = tiny_bert(positions, "meta")
    assert at in empty.to_empty(device=device)._constants


# --------------------------------------------------------------------------
# clipping around the exchange
# --------------------------------------------------------------------------

@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("stage", ["local", "reduced"])
def test_norms_of_steps_stay(device, stage):
    """Norms that are collected without a synchronisation and read at the end,
    before and after the exchange is captured."""
    gen = torch.Generator().manual_seed(6)
    torch.manual_seed(6)
    model = torch.nn.Linear(60, 40).to(device)
    opt = dr.DistributedOptimizer(torch.optim.SGD(model.parameters(), lr=0.0),
                                  make_grc(clip_norm=1e-3, clip_stage=stage,
                                           memory="none"), model)
    norms, want = [], []
    for step in range(9):
        x = torch.randn(5, 60, generator=gen).to(device)
        opt.zero_grad(set_to_none=False)
        (model(x).sum() * 2 ** step).backward()
        if stage == "local":
            want.append(global_norm(p.grad for p in model.parameters()))
        opt.step()
        norms.append(opt.last_grad_norm)
        if stage == "reduced":
            want.append(norms[-1].item())
    assert (opt._graph is not None) == (device == "cuda")
    assert len({n.data_ptr() for n in norms}) == len(norms)
    for a, c in zip(norms, want):
        assert abs(a.item() - c) <= 1e-6 * c
    assert norms[-1].item() > 50 * norms[0].item()
