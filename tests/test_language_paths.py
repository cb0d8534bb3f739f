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


def rank_main(rank, world, port, work, queue):
    """Runs work(rank) in a process group over the loopback address."""
    import os
    import traceback

    import torch.distributed as dist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.set_num_threads(1)
    try:
        dist.init_process_group("gloo", rank=rank, world_size=world)
        queue.put((rank, work(rank), None))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:  # noqa: BLE001
        queue.put((rank, None, traceback.format_exc()[-1500:]))


def run_ranks(world, work):
    """What work(rank) returned (plain values) on each of `world` ranks."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    procs = [ctx.Process(target=rank_main, args=(r, world, port, work, queue))
             for r in range(world)]
    for p in procs:
        p.start()
    results = {}
    for _ in procs:
        rank, value, error = queue.get(timeout=240)
        assert error is None, error
        results[rank] = value
    for p in procs:
        p.join(timeout=60)
    return [results[r] for r in range(world)]


def clipped_exchange(rank, stage, way):
    """[largest deviation from clipping by hand, this rank's norm, the norm
    that the first step should have], after two steps on this rank's data."""
    from deepreduce_amd.optimizer import reduce_gradients

    torch.manual_seed(9)
    bound = 0.5
    models = [torch.nn.Sequential(torch.nn.Linear(60, 80), torch.nn.Tanh(),
                                  torch.nn.Linear(80, 50)) for _ in range(2)]
    models[1].load_state_dict(models[0].state_dict())
    grcs = [make_grc(clip_norm=bound, clip_stage=stage), make_grc()]
    reducers = [OverlappedReducer(m, g) for m, g in zip(models, grcs)] if way == "overlapped" \
        else [None, None]
    gen = torch.Generator().manual_seed(100 + rank)
    worst, norms = 0.0, []
    for step in range(2):
        x = torch.randn(16, 60, generator=gen)
        for model in models:
            model.zero_grad()
            (model(x) ** 2).sum().backward()
        grads = [p.grad for p in models[1].parameters()]

        def by_hand():
            norm = global_norm(grads)
            for g in grads:
                g.mul_(min(1.0, bound / norm))
            return norm

        before = by_hand() if stage == "local" else None
        for model, grc, reducer in zip(reversed(models), reversed(grcs), reversed(reducers)):
            if reducer:
                reducer.finalize()
            else:
                reduce_gradients(model, grc, fused=way == "fused")
        before = by_hand() if stage == "reduced" else before
        norms.append((grcs[0].last_grad_norm.item(), before))
        for p, q in zip(models[0].parameters(), models[1].parameters()):
            worst = max(worst, (p.grad - q.grad).abs().max().item())
    return worst, norms


def local_fused(rank):
    return clipped_exchange(rank, "local", "fused")


def local_by_tensor(rank):
    return clipped_exchange(rank, "local", "by tensor")


def reduced_fused(rank):
    return clipped_exchange(rank, "reduced", "fused")


def reduced_overlapped(rank):
    return clipped_exchange(rank, "reduced", "overlapped")


@pytest.mark.timeout(300)
@pytest.mark.parametrize("work", [local_fused, local_by_tensor, reduced_fused,
                                  reduced_overlapped], ids=lambda w: w.__name__)
def test_two_ranks_clip(work):
    """Each rank its own gradients before the exchange, all the same ones after
    it, against the same steps clipped by hand."""
    results = run_ranks(2, work)
    for worst, norms in results:
        # a product rounded to 32 bits once more, of values of at most the bound
        assert worst <= 1e-6 * 0.5
        for got, want in norms:
            assert want > 0.5 and abs(got - want) <= 1e-6 * want
    first, second = ([n for n, _ in r[1]] for r in results)
    assert (first == second) == work.__name__.startswith("reduced")


def federated_rank(rank):
    """One round of one local step: the norms of what this rank compressed, and
    of how far the server's model went."""
    from deepreduce_amd.federated_dist import FederatedDistRunner

    torch.manual_seed(10)
    model = torch.nn.Linear(30, 10)
    start = [p.detach().clone() for p in model.parameters()]
    compressor, seen = make_grc(compress_ratio=1.0).compressor, []
    compress = compressor.compress
    compressor.compress = lambda t, n: (seen.append(t.clone()), compress(t, n))[1]
    runner = FederatedDistRunner(model, compressor, local_lr=0.5, clip_norm=0.1)
    runner.memory = dr.NoneMemory()
    gen = torch.Generator().manual_seed(rank)
    x, y = torch.randn(12, 30, generator=gen) * 50, torch.randint(0, 10, (12,), generator=gen)
    runner.round(lambda: [(x, y)])
    moved = [p.detach() - s for p, s in zip(model.parameters(), start)]
    return global_norm(seen), global_norm(moved)


@pytest.mark.timeout(300)
def test_federated_ranks_clip():
    (sent, moved), (client, also), (other, _) = run_ranks(3, federated_rank)
    # what a client sends is its one step's gradient, clipped; 32-bit rounding
    # of the parameters, of size 0.2 or less, shows in the difference of two
    assert abs(client - 0.1) <= 1e-4 and abs(other - 0.1) <= 1e-4
    assert sent == 0 and moved == also and 0 < moved <= 0.1 + 1e-4
