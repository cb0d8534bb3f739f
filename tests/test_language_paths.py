"""The language-model operators in the framework's own paths, where a program
leaves the usual order of steps: evaluation before training, parameters of
other types, steps without gradients, more than one rank."""
import copy
import math

import pytest
import torch

import deepreduce_amd as dr
from deepreduce_amd import ops
from deepreduce_amd.parallel import OverlappedReducer
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


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16], ids=str)
@pytest.mark.parametrize("way", ["local", "reduced", "overlapped"])
def test_clip_of_parameters_of_other_types(device, dtype, way):
    """Parameters in 64 and 16 bits beside some in 32 clip at every stage."""
    from deepreduce_amd.optimizer import reduce_gradients

    torch.manual_seed(7)
    model = torch.nn.Sequential(torch.nn.Linear(40, 60), torch.nn.Linear(60, 50)).to(device)
    model[1].to(dtype)
    grc = dr.deepreduce_from_params({
        "compressor": "none", "memory": "none", "communicator": "allgather", "clip_norm": 0.25,
        "clip_stage": "local" if way == "local" else "reduced"})
    reducer = OverlappedReducer(model, grc) if way == "overlapped" else None
    x = torch.randn(8, 40, device=device)
    model[1](model[0](x).to(dtype)).float().square().sum().backward()
    before = [p.grad.double().clone() for p in model.parameters()]
    if reducer:
        reducer.finalize()
    else:
        reduce_gradients(model, grc)
    norm = global_norm(before)
    # a gradient is rounded to its type once or twice
    u = torch.finfo(dtype).eps if dtype == torch.bfloat16 else 2.0 ** -22
    assert norm > 1 and abs(grc.last_grad_norm.item() - norm) <= u * norm
    for p, b in zip(model.parameters(), before):
        assert p.grad.dtype == p.dtype
        assert (p.grad.double() - b * 0.25 / norm).abs().max() <= u * 0.25


# --------------------------------------------------------------------------
# federated clients and several ranks
# --------------------------------------------------------------------------

def test_federated_step_without_gradients():
    """A step that leaves no parameter a gradient has nothing to clip."""
    from deepreduce_amd.federated import FederatedClient, FederatedServer

    torch.manual_seed(8)
    compressor = make_grc().compressor
    model = torch.nn.Linear(30, 20)
    for p in model.parameters():
        p.requires_grad_(False)
    x = torch.randn(4, 30, requires_grad=True)
    sent = []
    for bound in (None, 0.1):
        server = FederatedServer(model, compressor)
        client = FederatedClient(model, compressor, clip_norm=bound)
        sent.append(client.round(server.broadcast_payload(), lambda: [(x, None)],
                                 loss_fn=lambda out, y: out.square().sum()))
    for name, (payload, _) in sent[0].items():
        for a, c in zip(payload, sent[1][name][0]):
            assert torch.equal(a, c)
