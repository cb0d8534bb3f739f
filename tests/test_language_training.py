"""The language-model operators in the framework's own paths: BERT on packed
rows, gradient clipping before and after the compressed exchange, federated
clients that clip their local steps."""
import math

import pytest
import torch

import deepreduce_amd as dr
from deepreduce_amd import ops
from deepreduce_amd.federated import FederatedClient, FederatedServer
from deepreduce_amd.models.bert import BertBase, document_positions
from deepreduce_amd.parallel import OverlappedReducer

BOTH = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
POSITIONS = ["learned", "rotary", "distance"]


def tiny_bert(positions="learned", device="cpu"):
    torch.manual_seed(0)
    return BertBase(vocab=97, hidden=64, layers=2, heads=4, ffn=128, max_len=96,
                    positions=positions).to(device)


def test_document_positions():
    documents = torch.tensor([[5, 5, 5, 2, 2, -1, -1, -1], [0, 1, 1, 0, 0, 0, 3, 3]],
                             dtype=torch.int32)
    assert document_positions(documents).tolist() == [[0, 1, 2, 0, 1, 0, 1, 2],
                                                      [0, 0, 1, 0, 1, 2, 0, 1]]


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("positions", POSITIONS)
def test_bert_packed_rows_are_their_documents(device, positions):
    """Logits and parameter gradients of two packed rows against the same
    documents one by one, in 32 bits."""
    model = tiny_bert(positions, device)
    lengths = [[30, 1, 45], [70]]
    ids, documents, parts = [], [], []
    gen = torch.Generator().manual_seed(1)
    for row in lengths:
        tokens = [torch.randint(0, 97, (n,), generator=gen) for n in row]
        pad = 80 - sum(row)
        parts += tokens
        ids.append(torch.cat(tokens + [torch.zeros(pad, dtype=torch.int64)]))
        documents.append(torch.cat([torch.full((n,), i, dtype=torch.int32)
                                    for i, n in enumerate(row)]
                                   + [torch.full((pad,), -1, dtype=torch.int32)]))
    ids, documents = torch.stack(ids).to(device), torch.stack(documents).to(device)
    out = model(ids, documents)
    (out[documents >= 0].float() ** 2).sum().backward()
    packed = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    alone = torch.cat([model(t.unsqueeze(0).to(device))[0] for t in parts])
    (alone.float() ** 2).sum().backward()
    # two layers of sums of 64 to 128 products in 32 bits, in other orders
    assert (out[documents >= 0] - alone).abs().max() <= 1e-5 * alone.abs().max()
    for n, p in model.named_parameters():
        assert (packed[n] - p.grad).abs().max() <= 1e-4 * p.grad.abs().max() + 1e-6, n


def test_bert_keeps_its_default():
    """Whole rows with learned positions: the state and results of before."""
    model = tiny_bert()
    assert "pos.weight" in model.state_dict()
    assert "pos.weight" not in tiny_bert("rotary").state_dict()
    ids = torch.randint(0, 97, (2, 40))
    whole = model(ids, torch.zeros(2, 40, dtype=torch.int32))
    assert (model(ids) - whole).abs().max() <= 1e-5 * whole.abs().max()
    with pytest.raises(ValueError):
        model(torch.zeros(1, 97, dtype=torch.int64))
    assert tiny_bert("distance")(torch.zeros(1, 97, dtype=torch.int64)).shape == (1, 97, 97)
    with pytest.raises(ValueError):
        BertBase(positions="other")


def make_grc(**more):
    return dr.deepreduce_from_params({
        "compressor": "topk", "memory": "residual", "communicator": "allgather",
        "compress_ratio": 0.05, "deepreduce": "index", "index": "bloom", "policy": "leftmost",
        **more})


def global_norm(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def clip(grads, bound):
    factor = min(1.0, bound / global_norm(grads))
    return [(g.double() * factor).float() for g in grads]


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("stage", ["local", "reduced"])
@pytest.mark.parametrize("fused", [True, False])
def test_clip_around_the_exchange(device, stage, fused):
    """Steps with clip_norm against the same steps with the gradients clipped
    by hand before or after an exchange without it."""
    from deepreduce_amd.optimizer import reduce_gradients

    bound = 0.5
    models = [torch.nn.Sequential(torch.nn.Linear(60, 80), torch.nn.Tanh(),
                                  torch.nn.Linear(80, 50)).to(device) for _ in range(2)]
    models[1].load_state_dict(models[0].state_dict())
    grcs = [make_grc(clip_norm=bound, clip_stage=stage), make_grc()]
    gen = torch.Generator().manual_seed(2)
    for step in range(3):
        x = torch.randn(16, 60, generator=gen).to(device)
        for model in models:
            model.zero_grad()
            (model(x) ** 2).sum().backward()
        grads = [p.grad for p in models[1].parameters()]
        if stage == "local":
            before = global_norm(grads)
            for g, c in zip(grads, clip(grads, bound)):
                g.copy_(c)
        reduce_gradients(models[1], grcs[1], fused=fused)
        if stage == "reduced":
            before = global_norm(grads)
            for g, c in zip(grads, clip(grads, bound)):
                g.copy_(c)
        reduce_gradients(models[0], grcs[0], fused=fused)
        assert abs(grcs[0].last_grad_norm.item() - before) <= 1e-6 * before
        for p, q in zip(models[0].parameters(), models[1].parameters()):
            assert (p.grad - q.grad).abs().max() <= 1e-6 * bound
        if stage == "reduced":
            assert global_norm(p.grad for p in models[0].parameters()) <= bound * (1 + 1e-6)


def test_clip_options():
    with pytest.raises(ValueError):
        make_grc(clip_norm=0.0)
    with pytest.raises(ValueError):
        make_grc(clip_norm=-1)
    with pytest.raises(ValueError):
        make_grc(clip_norm="1")
    with pytest.raises(ValueError):
        make_grc(clip_stage="local")
    with pytest.raises(ValueError):
        make_grc(clip_norm=1.0, clip_stage="other")
    model = torch.nn.Linear(40, 40)
    with pytest.raises(ValueError):
        OverlappedReducer(model, make_grc(clip_norm=1.0))
    opt = dr.DistributedOptimizer(torch.optim.SGD(model.parameters(), lr=0.1), make_grc(), model)
    assert opt.last_grad_norm is None


@pytest.mark.parametrize("device", BOTH)
def test_overlapped_reducer_clips(device):
    torch.manual_seed(3)
    model = torch.nn.Sequential(torch.nn.Linear(50, 60), torch.nn.Linear(60, 40)).to(device)
    grc = make_grc(clip_norm=0.25, clip_stage="reduced")
    reducer = OverlappedReducer(model, grc)
    (model(torch.randn(8, 50, device=device)) ** 2).sum().backward()
    reducer.finalize()
    assert grc.last_grad_norm.item() > 0.25
    norm = global_norm([p.grad for p in model.parameters()])
    assert abs(norm - 0.25) <= 1e-6


@pytest.mark.parametrize("device", BOTH)
def test_federated_client_clips(device):
    torch.manual_seed(4)
    model = torch.nn.Linear(30, 10).to(device)
    compressor = make_grc().compressor
    server = FederatedServer(model, compressor)
    x, y = torch.randn(12, 30, device=device) * 50, torch.randint(0, 10, (12,), device=device)
    for bound in (0.1, 1e9):
        client = FederatedClient(model, compressor, local_lr=0.5, clip_norm=bound)
        client.c2s_memory = dr.NoneMemory()
        seen = []
        client.compressor = type("Record", (), {
            "compress": lambda self, t, n: (seen.append(t.clone()), compressor.compress(t, n))[1],
            "decompress": lambda self, p, c: compressor.decompress(p, c)})()
        client.round(server.broadcast_payload(), lambda: [(x, y)])
        # one step: what the client sends is its clipped gradient
        norm = global_norm(seen)
        assert abs(norm - 0.1) <= 1e-3 if bound == 0.1 else norm > 1


@pytest.mark.gpu
@pytest.mark.parametrize("stage", ["local", "reduced"])
def test_packed_bert_step_replays(stage):
    """Whole steps of a packed BERT with rotary positions, clipped and
    exchanged: the captured exchange against the eager one, step by step."""
    results = []
    for use_graph in (False, True):
        model = tiny_bert("rotary", "cuda")
        grc = make_grc(clip_norm=0.05, clip_stage=stage)
        opt = dr.DistributedOptimizer(torch.optim.SGD(model.parameters(), lr=0.5), grc, model,
                                      use_graph=use_graph)
        documents = torch.tensor([[0] * 30 + [1] * 40 + [-1] * 10, [0] * 80],
                                 dtype=torch.int32, device="cuda")
        norms = []
        for step in range(8):
            gen = torch.Generator().manual_seed(step)
            ids = torch.randint(0, 97, (2, 80), generator=gen).cuda()
            opt.zero_grad(set_to_none=False)
            out = model(ids, documents)
            torch.nn.functional.cross_entropy(
                out.flatten(0, 1).float(),
                torch.where(documents >= 0, ids.roll(1, 1), -100).flatten()).backward()
            opt.step()
            norms.append(opt.last_grad_norm.item())
        assert (opt._graph is not None) == use_graph
        results.append((norms, [p.detach().clone() for p in model.parameters()]))
    assert results[0][0][0] > 0.05  # the first step at least is clipped
    for a, c in zip(results[0][0], results[1][0]):
        assert abs(a - c) <= 1e-4 * a
    for a, c in zip(results[0][1], results[1][1]):
        assert (a - c).abs().max() <= 1e-3 * a.abs().max()


@pytest.mark.gpu
def test_operators_together_follow_64_bits():
    """Rotary, attention on documents with a distance bias, and the clipped
    gradients of a projection, in bfloat16 against 64 bits."""
    b, s, h, d = 2, 130, 3, 64
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(b, s, 96, generator=gen).bfloat16()
    weight = (torch.randn(3 * h * d, 96, generator=gen) / 10).bfloat16()
    documents = torch.tensor([[0] * 50 + [1] * 60 + [-1] * 20, [0] * 130], dtype=torch.int32)
    positions = document_positions(documents)
    slopes = torch.tensor([0.5, 0.1, 0.02])
    frequencies = ops.rotary_frequencies(d)

    w = weight.cuda().requires_grad_(True)
    q, k, v = (x.cuda() @ w.t()).view(b, s, 3, h, d).unbind(2)
    q, k = ops.rotary(q, k, positions.cuda(), frequencies.cuda())
    out = ops.attention(q, k, v, documents.cuda(), slopes.cuda())
    (grad,) = torch.autograd.grad(out.float().square().sum(), w)
    (clipped,), norm = ops.clip_grad_norm([grad], 1.0, dtype=torch.float32)

    w = weight.double().requires_grad_(True)
    q, k, v = (x.double() @ w.t()).view(b, s, 3, h, d).unbind(2)
    angle = positions.double()[..., None, None] * frequencies

    def turn(t):
        first, second = t[..., :d // 2], t[..., d // 2:]
        return torch.cat((first * angle.cos() - second * angle.sin(),
                          first * angle.sin() + second * angle.cos()), -1)

    at = torch.arange(s)
    scores = torch.einsum("bihd,bjhd->bhij", turn(q), turn(k)) * d ** -0.5
    scores = scores - slopes.double().view(1, h, 1, 1) * (at[:, None] - at[None]).abs()
    seen = ((documents[:, :, None] == documents[:, None]) & (documents[:, None] >= 0))[:, None]
    scores = scores.masked_fill(~seen, -1e300)
    p = torch.softmax(scores, -1) * seen
    want = torch.einsum("bhij,bjhd->bihd", p, v)
    (exact,) = torch.autograd.grad(want.square().sum(), w)
    # five roundings to bfloat16 one after the other (the projection, rotary,
    # probabilities, the output and the gradients), each of half a step, in root
    # mean square, doubled for their growth through the softmax
    tol = 2 * 5 * torch.finfo(torch.bfloat16).eps / 2
    assert (out.double().cpu() - want).norm() <= tol * want.norm()
    assert (grad.double().cpu() - exact).norm() <= tol * exact.norm()
    assert abs(norm.item() - exact.norm().item()) <= tol * exact.norm().item()
    assert abs(clipped.norm().item() - 1.0) <= 1e-5
