"""Attention over packed documents, rotary positions, gradient norm and
clipping: every path against the formulas in 64 bits.

Tolerances are computed beside each expected value from the roundings that a
path makes: u = eps / 2 of the type for each rounding to it, E = 2^-24 for
each operation in 32 bits.
"""
import math

import pytest
import torch

from deepreduce_amd import ops

E = 2.0 ** -24
BOTH = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    off = torch.where(want.isnan(), torch.zeros_like(want), (got - want).abs() - tol)
    if off.numel() == 0:
        return
    worst = off.argmax()
    assert off.max() <= 0, (f"{what}: {got.flatten()[worst]} for {want.flatten()[worst]}, "
                            f"tolerance {tol.flatten()[worst]}")


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def seen_pairs(documents, causal, b, sq, sk):
    p = torch.arange(sk - sq, sk).unsqueeze(1)
    j = torch.arange(sk).unsqueeze(0)
    seen = torch.ones(b, sq, sk, dtype=torch.bool)
    if causal:
        seen &= j <= p
    if documents is not None:
        d = documents.cpu()
        seen &= (d[:, sk - sq:, None] == d[:, None, :]) & (d >= 0)[:, None, :]
    return seen, (p - j).abs()


def attention_oracle(q, k, v, documents, slopes, causal, scale, dout=None):
    """{name: (value, tolerance)} in 64 bits.  What is hidden is set to zero
    before any product, so that it cannot reach one."""
    dtype = q.dtype
    u = half_step(dtype)
    b, sq, hq, d = q.shape
    sk, hkv = k.shape[1:3]
    group = hq // hkv
    seen, far = seen_pairs(documents, causal, b, sq, sk)
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    shapes = {"out": q.shape}
    if dout is not None:
        shapes.update(dq=q.shape, dk=k.shape, dv=v.shape)
        dout = dout.detach().double().cpu()
    res = {n: (torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64))
           for n, s in shapes.items()}

    def put(name, where, value, tol):
        res[name][0][where] += value
        res[name][1][where] += tol

    def product(w, x, s):  # w @ x over pairs in s only
        bad = ~torch.isfinite(x)
        if not bad.any():
            return w @ x
        y = w @ x.masked_fill(bad, 0.0)
        for j in range(x.shape[0]):
            if bad[j].any():
                term = w[:, j:j + 1] * x[j].masked_fill(~bad[j], 0.0)
                y = y + torch.where(s[:, j:j + 1], term, torch.zeros_like(term))
        return y

    for e in range(b):
        s_e = seen[e]
        for h in range(hq):
            g = h // group
            Q, K, V = q[e, :, h], k[e, :, g], v[e, :, g]
            s = scale * (Q @ K.T)
            bias = far * float(slopes[h]) if slopes is not None else torch.zeros_like(s)
            s = (s - bias).masked_fill(~s_e, -math.inf)
            top = s.amax(1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            w = torch.exp(s - top)
            total = w.sum(1, keepdim=True)
            P = torch.where(s_e, w / torch.where(total == 0, 1.0, total), 0.0)
            # a score is off by its d products and sums, the scaling and the
            # bias; exp turns that into a relative error of P, and so does the
            # row's sum, which is off by no more than its worst score
            es = (d + 8) * E * (abs(scale) * (Q.abs() @ K.abs().T) + 4 * bias) \
                + 4 * E * torch.where(s_e, s.abs() + top.abs(), 0.0) + 8 * E
            es = torch.where(s_e, es, 0.0)
            rel = es + es.amax(1, keepdim=True) + (sk + 8) * E
            O = product(P, V, s_e)
            # in 16 bits P is rounded before its product with V.  Where that
            # has no normal numbers left it is off by a fixed step instead:
            # 2^-126, the least float, which may be flushed, and in fp16 half
            # of 2^-24 after a scaling by 2^12 (the row's sum is 1 or more)
            half = 0.0 if dtype == torch.float32 else u
            floor = 2.0 ** -37 if dtype == torch.float16 else 2.0 ** -125
            to = product(torch.where(s_e, P * (rel + half + (sk + 8) * E) + floor, 0.0),
                         V.abs(), s_e) * 1.01 + u * O.abs()
            tiny = torch.finfo(dtype).tiny * 2  # values below the type's range
            put("out", (e, slice(None), h), O, to + tiny)
            if dout is None:
                continue
            dO = dout[e, :, h]
            dP = torch.where(s_e, dO @ V.T, 0.0)
            delta = torch.where(s_e.any(1), (dO * O).sum(1), 0.0).unsqueeze(1)
            edelta = ((dO.abs() * (to + d * E * O.abs())).sum(1)).unsqueeze(1)
            edelta = torch.where(s_e.any(1, keepdim=True), edelta, 0.0)
            dS = torch.where(s_e, P * (dP - delta), 0.0)
            edP = torch.where(s_e, (d + 4) * E * (dO.abs() @ V.abs().T), 0.0)
            # dS has the same floor times its factor, in fp16 times the largest
            # dO (scaled to 1 and by 2^8 before the rounding, steps of 2^-24)
            least = (2.0 ** -33 * 2 * dO[torch.isfinite(dO)].abs().max()
                     if dtype == torch.float16 else floor * (1 + (dP - delta).abs()))
            edS = torch.where(s_e, P * (edP + edelta) * 1.1 + dS.abs() * (rel + half + 8 * E)
                              + least, 0.0)
            n = (max(sq * group, sk) + 8) * E
            back = s_e.T
            dq = scale * product(dS, K, s_e)
            put("dq", (e, slice(None), h), dq,
                abs(scale) * product(edS + n * dS.abs(), K.abs(), s_e) + u * dq.abs() + tiny)
            put("dk", (e, slice(None), g), scale * product(dS.T, Q, back),
                abs(scale) * product((edS + n * dS.abs()).T, Q.abs(), back) + tiny)
            put("dv", (e, slice(None), g), product(P.T, dO, back),
                product(torch.where(s_e, P * (rel + half + n) + floor, 0.0).T, dO.abs(), back)
                + tiny)
    for name in ("dk", "dv"):
        if name in res:
            res[name][1].add_(u * res[name][0].abs())
    return res


def pack(lengths, sk, pad=-1):
    row = [i for i, n in enumerate(lengths) for _ in range(n)]
    return row[:sk] + [pad] * (sk - len(row))


def attention_inputs(b, sq, sk, hq, hkv, d, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(device)  # noqa: E731
    return make(b, sq, hq, d), make(b, sk, hkv, d), make(b, sk, hkv, d), make(b, sq, hq, d)


def check_attention(q, k, v, dout, documents=None, slopes=None, causal=False, scale=None,
                    dq_of=None):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.attention(*leaves, documents=documents, slopes=slopes, causal=causal, scale=scale)
    plain = ops.attention(q, k, v, documents=documents, slopes=slopes, causal=causal, scale=scale)
    grads = torch.autograd.grad(out, leaves, dout)
    want = attention_oracle(q, k, v, documents, slopes, causal,
                            q.shape[-1] ** -0.5 if scale is None else scale, dout)
    assert out.dtype == q.dtype and out.shape == q.shape
    assert_within(out, *want["out"], "out")
    assert_within(plain, *want["out"], "out without gradients")
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert_within(got, *want[name], name)


DOCS = {
    "none": lambda b, s: None,
    # several documents, a break inside each tile, padding at the end of odd rows
    "packed": lambda b, s: torch.tensor(
        [pack([max(1, s // 3), 1, max(1, s // 4), s], s if e % 2 == 0 else max(1, s - s // 5))
         + [-1] * (0 if e % 2 == 0 else s - max(1, s - s // 5)) for e in range(b)],
        dtype=torch.int32),
    # documents that alternate token by token
    "mixed": lambda b, s: torch.arange(s, dtype=torch.int32).remainder(3).sub(
        (torch.arange(s) % 5 == 4).int() * 9).repeat(b, 1),
    # nothing but padding in one row, one visible token in the others
    "empty": lambda b, s: torch.tensor(
        [[-1] * s if e == 0 else [-1] * (s - 1) + [7] for e in range(b)], dtype=torch.int32),
}

SHAPES = [  # b, sq, sk, hq, hkv, d
    (1, 1, 1, 1, 1, 8),
    (2, 16, 16, 2, 1, 16),
    (2, 65, 65, 3, 3, 64),
    (1, 130, 130, 4, 2, 40),
    (2, 1, 300, 6, 2, 64),
    (1, 3, 257, 4, 1, 128),
    (1, 100, 193, 2, 2, 80),
    (1, 257, 257, 2, 1, 128),
    (3, 33, 64, 2, 2, 96),
]


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("docs", list(DOCS))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention(device, dtype, shape, docs):
    b, sq, sk, hq, hkv, d = shape
    q, k, v, dout = attention_inputs(*shape, dtype, device, seed=sum(shape))
    documents = DOCS[docs](b, sk)
    documents = None if documents is None else documents.to(device)
    for causal in (False, True):
        slopes = torch.linspace(0.5, 0.01, hq).to(device) if causal == (d == 64) else None
        check_attention(q, k, v, dout, documents, slopes, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1000, 1000, 2, 1, 64), (1, 700, 1111, 2, 2, 128),
                                   (2, 1, 5003, 4, 2, 64), (1, 7, 2049, 3, 1, 32),
                                   (1, 45, 3001, 4, 2, 96), (40, 2, 131, 12, 4, 128)], ids=str)
def test_attention_long(dtype, shape):
    b, sq, sk, hq, hkv, d = shape
    q, k, v, dout = attention_inputs(*shape, dtype, "cuda", seed=sum(shape))
    documents = torch.tensor([pack([17, 400, 64, 1, 300, 5000], sk)] * b,
                             dtype=torch.int32, device="cuda")
    check_attention(q, k, v, dout, documents)
    check_attention(q, k, v, dout, causal=True,
                    slopes=torch.linspace(0.1, 0.0, hq, device="cuda"))
    check_attention(q, k, v, dout, scale=0.7)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_strides(device, dtype):
    """Slices of one projection, heads before positions, an expanded gradient
    and addresses that are no multiple of 16 bytes."""
    b, s, h, d = 2, 70, 4, 64
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(b, s, 3, h, d, generator=gen).to(dtype).to(device)
    q, k, v = qkv.unbind(2)
    dout = torch.randn(1, 1, h, d, generator=gen).to(dtype).to(device).expand(b, s, h, d)
    documents = DOCS["packed"](b, s).to(device)
    check_attention(q, k, v, dout, documents)
    q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    check_attention(q, k, v, dout, documents[:, :].t().contiguous().t(), causal=True)
    flat = torch.randn(b * s * h * d + 1, generator=gen).to(dtype).to(device)[1:]
    check_attention(flat.view(b, s, h, d), k, v, dout)
    check_attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, dout)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, "lowest"], ids=str)
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_attention_keeps_what_is_hidden(device, dtype, bad, which):
    """A document with infinities, NaN or the type's lowest value changes no
    other document, nor does padding: not the results, not the gradients."""
    b, s, hq, hkv, d = 1, 150, 2, 1, 64
    clean = dict(zip(("q", "k", "v", "dout"), attention_inputs(b, s, s, hq, hkv, d, dtype,
                                                               device, seed=3)))
    documents = torch.tensor([pack([40, 70, 30], 140) + [-1] * 10], dtype=torch.int32,
                             device=device)
    value = torch.finfo(dtype).min if bad == "lowest" else bad
    dirty = {n: t.clone() for n, t in clean.items()}
    dirty[which][:, 45] = value
    dirty[which][:, 145] = value
    results = []
    for x in (clean, dirty):
        leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v")]
        out = ops.attention(*leaves, documents=documents)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, x["dout"])])
    keep = torch.ones(s, dtype=torch.bool, device=device)
    keep[40:110] = False
    for name, a, c in zip(("out", "dq", "dk", "dv"), *results):
        assert torch.isfinite(c[:, keep]).all(), name
        # a guarded tile may add in another order
        scale = a.float().abs().max()
        assert (a[:, keep].float() - c[:, keep].float()).abs().max() <= \
            4 * (half_step(dtype) + 256 * E) * scale, name
        assert not c[:, 140:].any(), name
    if bad != "lowest" and which != "dout":
        assert not torch.isfinite(results[1][0][:, 40:110]).all()


@pytest.mark.parametrize("device", BOTH)
def test_attention_causal_keeps_the_future(device):
    q, k, v, _ = attention_inputs(1, 100, 100, 2, 2, 32, torch.float32, device)
    a = ops.attention(q, k, v, causal=True)
    k[:, 60:], v[:, 60:] = math.nan, math.inf
    c = ops.attention(q, k, v, causal=True)
    assert (a[:, :60] - c[:, :60]).abs().max() <= 256 * E * a.abs().max()
    assert c[:, 60:].isnan().all()


@pytest.mark.parametrize("device", BOTH)
def test_attention_large_scores(device):
    """Scores of hundreds: the running maximum carries them."""
    q, k, v, dout = attention_inputs(1, 90, 90, 2, 2, 64, torch.float32, device)
    check_attention(q * 10, k * 10, v, dout)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_attention_scale(device, dtype, scale):
    q, k, v, dout = attention_inputs(1, 75, 75, 2, 1, 64, dtype, device)
    documents = DOCS["packed"](1, 75).to(device)
    check_attention(q, k, v, dout, documents, torch.tensor([0.2, 0.0], device=device), True, scale)
    check_attention(q[:, -1:], k, v, dout[:, -1:], documents, None, True, scale)


@pytest.mark.parametrize("device", BOTH)
def test_attention_without_rows(device):
    for b, sq, sk in ((0, 4, 4), (2, 0, 5), (2, 0, 0)):
        q, k, v, dout = attention_inputs(b, sq, sk, 2, 1, 16, torch.float32, device)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = ops.attention(*leaves)
        assert out.shape == q.shape
        for g, t in zip(torch.autograd.grad(out, leaves, dout), leaves):
            assert g.shape == t.shape and not g.any()


def test_attention_differences():
    """The CPU path's gradients against differences of its results."""
    q, k, v, dout = attention_inputs(1, 6, 9, 2, 1, 8, torch.float32, "cpu")
    documents = torch.tensor([pack([4, 3], 7) + [-1, 1]], dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    f = lambda *x: (ops.attention(*x, documents=documents,  # noqa: E731
                                  slopes=torch.tensor([0.3, 0.1])) * dout).sum()
    grads = torch.autograd.grad(f(*leaves), leaves)
    step = 1e-2
    for n, g in enumerate(grads):
        way = torch.randn(g.shape, generator=torch.Generator().manual_seed(n))
        ends = [f(*[t.detach() + (sign * step * way if m == n else 0)
                    for m, t in enumerate(leaves)]) for sign in (1, -1)]
        # third derivatives times step^2 / 6, and the rounding of the difference
        assert abs((ends[0] - ends[1]) / (2 * step) - (g * way).sum()) <= 2e-2 * g.norm() + 1e-3


@pytest.mark.parametrize("device", BOTH)
def test_attention_refuses(device):
    q, k, v, _ = attention_inputs(2, 8, 8, 4, 2, 16, torch.float32, device)
    docs = torch.zeros(2, 8, dtype=torch.int32, device=device)
    slopes = torch.zeros(4, device=device)
    wrong = [
        dict(q=q[0]), dict(q=q.double()), dict(k=k.half()), dict(v=v[:, :7]), dict(k=k[:1], v=v[:1]),
        dict(k=k[:, :7], v=v[:, :7]), dict(q=q[:, :, :3]),
        dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]),
        dict(documents=docs.long()), dict(documents=docs[:, :7]), dict(documents=docs[:1]),
        dict(slopes=slopes.double()), dict(slopes=slopes[:3]), dict(scale=math.nan),
        dict(slopes=slopes.clone().requires_grad_(True)),
        dict(q=torch.zeros(2, 8, 4, 136, device=device), k=torch.zeros(2, 8, 2, 136, device=device),
             v=torch.zeros(2, 8, 2, 136, device=device)),
    ]
    if device == "cuda":
        wrong += [dict(k=k.cpu()), dict(documents=docs.cpu()), dict(slopes=slopes.cpu())]
    for change in wrong:
        with pytest.raises(ValueError):
            ops.attention(**{**dict(q=q, k=k, v=v), **change})


@pytest.mark.parametrize("device", BOTH)
def test_attention_document_numbers(device):
    """Any number names a document: the largest, zero, far apart; every
    negative one is padding."""
    q, k, v, dout = attention_inputs(1, 100, 100, 2, 2, 32, torch.float32, device)
    top, least = 2 ** 31 - 1, -2 ** 31
    row = [top] * 20 + [least] * 10 + [0] * 30 + [-1] * 5 + [top] * 10 + [-7] * 5 + [least + 1] * 20
    documents = torch.tensor([row], dtype=torch.int32, device=device)
    check_attention(q, k, v, dout, documents)
    check_attention(q[:, 75:76], k, v, dout[:, 75:76], documents, causal=True)
    out = ops.attention(q, k, v, documents)
    assert not out[0, 20:30].any() and not out[0, 60:65].any() and not out[0, 75:].any()


@pytest.mark.gpu
def test_attention_far_offsets():
    """A cache of over 2^31 values, of which the queries see the last rows, and
    rows that lie over 16 MB apart."""
    d, h, sq, near = 128, 32, 256, 300
    sk = 2 ** 19 + near
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.zeros(1, sk, h, d, dtype=torch.float16, device="cuda") for _ in range(2))
    for t in (k, v):
        t[:, -near:] = torch.randn(1, near, h, d, generator=gen, device="cuda").half()
    documents = torch.zeros(1, sk, dtype=torch.int32, device="cuda")
    documents[:, -near:] = 3
    for rows in (sq, 1):
        q, dout = (torch.randn(1, rows, h, d, generator=gen, device="cuda").half()
                   for _ in range(2))
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops.attention(*leaves, documents=documents, causal=True)
        dq, dk, dv = torch.autograd.grad(out, leaves, dout)
        few = [t.detach().clone().requires_grad_(True) for t in (q, k[:, -near:], v[:, -near:])]
        want = ops.attention(*few, causal=True)
        grads = torch.autograd.grad(want, few, dout)
        # the same sums in tiles that begin elsewhere
        for a, c in zip((out, dq, dk[:, -near:], dv[:, -near:]), (want, *grads)):
            assert (a.float() - c.float()).abs().max() <= 4 * 2.0 ** -11 * c.float().abs().max()
        assert not dk[:, :-near].any() and not dv[:, :-near].any()
        del out, dq, dk, dv, leaves
    del k, v
    wide = torch.randn(5, 9_000_000, generator=gen, device="cuda").half()
    k = wide[:, :64].view(1, 5, 1, 64)
    assert k.stride(1) * 2 > 1 << 24
    q, dout = (torch.randn(1, 5, 1, 64, generator=gen, device="cuda").half() for _ in range(2))
    check_attention(q, k, k, dout)


@pytest.mark.parametrize("device", BOTH)
def test_differentiable_once(device):
    q, k, v, dout = attention_inputs(1, 9, 9, 2, 1, 16, torch.float32, device)
    positions = torch.arange(9, device=device)
    frequencies = ops.rotary_frequencies(16, device=device)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    x, y = ops.rotary(q, k, positions, frequencies)
    out = ops.attention(x, y, v, causal=True)
    plain = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    again = torch.autograd.grad(out, leaves, dout, create_graph=True)
    for a, c in zip(plain, again):
        assert torch.equal(a, c)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(again[0].sum(), q)


@pytest.mark.gpu
def test_attention_repeats_and_replays():
    """Two eager calls, calls on another stream and every replay of a captured
    graph give the same bits, on inputs that change between the replays."""
    shape = (2, 200, 200, 4, 2, 64)
    documents = DOCS["packed"](2, 200).cuda()
    slopes = torch.linspace(0.5, 0.1, 4, device="cuda")
    static = [t.requires_grad_(i < 3) for i, t in
              enumerate(attention_inputs(*shape, torch.bfloat16, "cuda"))]

    def step(x):
        out = ops.attention(*x[:3], documents=documents, slopes=slopes, causal=True)
        return [out, *torch.autograd.grad(out, x[:3], x[3])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for seed in (1, 2, 3):
        fresh = attention_inputs(*shape, torch.bfloat16, "cuda", seed=seed)
        with torch.no_grad():
            for a, c in zip(static, fresh):
                a.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        eager = step([t.requires_grad_(i < 3) for i, t in enumerate(fresh)])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step(fresh)
        torch.cuda.current_stream().wait_stream(side)
        for a, c, e in zip(captured, eager, again):
            assert torch.equal(a, c) and torch.equal(c, e)


# --------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------

def rotary_oracle(x, positions, frequencies, interleaved, sign):
    u = half_step(x.dtype)
    y = x.detach().double().cpu()
    n = frequencies.numel()
    angle = positions.cpu().double()[..., None, None] * frequencies.cpu() * sign
    turn = torch.polar(torch.ones_like(angle), angle)
    first, second = ((slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved
                     else (slice(0, n), slice(n, 2 * n)))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous())
    want, tol = y.clone(), torch.zeros_like(y)
    r = z * turn
    want[..., first], want[..., second] = r.real, r.imag
    # sine and cosine are off by their own rounding and 4 E of the function,
    # the products and the sum by 3 E, the result by half a step
    size = z.real.abs() + z.imag.abs()
    for at, value in ((first, r.real), (second, r.imag)):
        tol[..., at] = 8 * E * size + u * (value.abs() + 8 * E * size) + 2 * torch.finfo(x.dtype).tiny
    return want, tol


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,hq,hkv,d,dim", [
    (1, 1, 1, 1, 8, 8), (2, 5, 3, 1, 64, 64), (1, 33, 4, 2, 40, 40), (2, 7, 2, 2, 128, 64),
    (1, 9, 2, 1, 66, 34), (3, 4, 1, 1, 10, 6), (1, 6, 2, 1, 64, 2), (1, 2500, 2, 1, 32, 32),
    (1, 3, 1, 1, 2, 2), (1, 2, 1, 1, 1024, 1024)])
def test_rotary(device, dtype, interleaved, b, s, hq, hkv, d, dim):
    gen = torch.Generator().manual_seed(s + d)
    make = lambda h: torch.randn(b, s, h, d, generator=gen).to(dtype).to(device)  # noqa: E731
    q, k, dq, dk = make(hq), make(hkv), make(hq), make(hkv)
    positions = torch.randint(-1000, 1_000_000, (b, s), generator=gen).to(device)
    frequencies = ops.rotary_frequencies(dim, factor=2.0, device=device)
    q.requires_grad_(True), k.requires_grad_(True)
    yq, yk = ops.rotary(q, k, positions, frequencies, interleaved)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    for got, x, sign in ((yq, q, 1), (yk, k, 1), (gq, dq, -1), (gk, dk, -1)):
        want, tol = rotary_oracle(x, positions, frequencies, interleaved, sign)
        assert got.dtype == dtype
        assert_within(got, want, tol, "rotary")
    # 32-bit positions of one row for all, and one side's gradient alone
    row = torch.arange(s, dtype=torch.int32, device=device)
    zq, zk = ops.rotary(q, k.detach(), row, frequencies, interleaved)
    assert_within(zk, *rotary_oracle(k, row.expand(b, s), frequencies, interleaved, 1), "k")
    (gq,) = torch.autograd.grad(zq, q, dq)
    assert_within(gq, *rotary_oracle(dq, row.expand(b, s), frequencies, interleaved, -1), "dq")


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rotary_strides(device, dtype, interleaved):
    gen = torch.Generator().manual_seed(0)
    qkv = torch.randn(2, 11, 3, 4, 64, generator=gen).to(dtype).to(device)
    flat = torch.randn(2 * 11 * 4 * 64 + 1, generator=gen).to(dtype).to(device)[1:]
    positions = torch.arange(11, device=device)
    frequencies = ops.rotary_frequencies(64, device=device)
    pairs = [qkv.unbind(2)[:2], (qkv[:, :, 0].transpose(1, 2).contiguous().transpose(1, 2),
                                 flat.view(2, 11, 4, 64)),
             (qkv[:, :, 0].transpose(2, 3).contiguous().transpose(2, 3), qkv[:, :, 1, :, :])]
    for q, k in pairs:
        for got, x in zip(ops.rotary(q, k, positions, frequencies, interleaved), (q, k)):
            assert got.is_contiguous()
            assert_within(got, *rotary_oracle(x, positions.expand(2, 11), frequencies,
                                              interleaved, 1), "rotary")


@pytest.mark.parametrize("device", BOTH)
def test_rotary_edges(device):
    frequencies = ops.rotary_frequencies(16, device=device)
    for b, s in ((0, 3), (2, 0)):
        q = torch.zeros(b, s, 2, 16, device=device)
        y, _ = ops.rotary(q, q, torch.zeros(s, dtype=torch.int64, device=device), frequencies)
        assert y.shape == q.shape
    q = torch.zeros(2, 3, 2, 16, device=device)
    at = torch.arange(3, device=device)
    for wrong in (dict(q=q[0]), dict(q=q.double(), k=q.double()), dict(k=q.half()),
                  dict(k=q[:, :2]), dict(positions=at.float()), dict(positions=at[:2]),
                  dict(positions=at.expand(3, 3)), dict(frequencies=frequencies.float()),
                  dict(frequencies=frequencies.repeat(2)), dict(frequencies=frequencies[:0]),
                  dict(frequencies=frequencies.clone().requires_grad_(True)),
                  dict(q=q[..., :15], k=q[..., :15])):
        with pytest.raises(ValueError):
            ops.rotary(**{**dict(q=q, k=q, positions=at, frequencies=frequencies), **wrong})


def test_rotary_frequencies():
    f = ops.rotary_frequencies(8, base=16.0)
    assert f.dtype == torch.float64 and f.tolist() == [1.0, 0.5, 0.25, 0.125]
    assert ops.rotary_frequencies(8, base=16.0, factor=4.0).tolist() == (f / 4).tolist()
    # by parts: 2 pi * 8 positions turn the pairs 8, 4, 2 and 1 times
    parts = ops.rotary_frequencies(8, base=16.0, factor=4.0, trained_length=50, low=2.0, high=6.0)
    turns = 50 * f / (2 * math.pi)
    kept = ((turns - 2) / 4).clamp(0, 1)
    assert torch.allclose(parts, f * kept + f / 4 * (1 - kept), rtol=1e-15, atol=0)
    assert parts[0] == f[0] and parts[3] == f[3] / 4
    for wrong in (dict(dim=7), dict(dim=0), dict(dim=8, base=1.0), dict(dim=8, factor=0.5),
                  dict(dim=8, trained_length=0), dict(dim=8, low=3.0, high=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**wrong)


# --------------------------------------------------------------------------
# gradient norm and clipping
# --------------------------------------------------------------------------

def gradients(kind, device, dtype):
    gen = torch.Generator().manual_seed(11)
    make = lambda *s: torch.randn(s, generator=gen).to(device)  # noqa: E731
    if kind == "one":
        return [make(1).to(dtype)]
    if kind == "odd":
        return [make(n).to(dtype) for n in (1, 3, 7, 0, 63, 64, 65, 1023, 4095, 4096, 4097, 20011)]
    if kind == "many":  # more than one table of them, types mixed
        return [make(1 + i % 37).to(TYPES[i % 3]) for i in range(300)]
    if kind == "views":  # parts of a bucket at odd offsets
        flat, at, got = make(9000).to(dtype), 1, []
        for n in (5, 1000, 1, 17, 4096, 2):
            got.append(flat[at:at + n])
            at += n
        return got
    if kind == "orders":  # channels last, transposed, gaps, one expanded
        return [make(4, 3, 5, 5).to(dtype).to(memory_format=torch.channels_last),
                make(8, 9).to(dtype).t(), make(6, 10).to(dtype)[:, :7],
                make(5).to(dtype).expand(4, 5), make(1, 9).to(dtype), make().to(dtype),
                make(8, 4, 1, 1).to(dtype).to(memory_format=torch.channels_last)]
    raise ValueError(kind)


KINDS = ["one", "odd", "many", "views", "orders"]


def norm_of(grads):
    return math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in grads))


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_grad_norm_and_clip(device, dtype, kind):
    grads = gradients(kind, device, dtype)
    want = norm_of(grads)
    norm = ops.grad_norm(grads)
    # the sum is in 64 bits, so the result is rounded to 32 bits once
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(norm.item() - want) <= 1.001 * E * want
    before = [g.clone() for g in grads]
    for bound in (want / 3, want * 2, 0.0, math.inf):
        factor = min(1.0, bound / want)
        for to in (None, *TYPES):
            outs, norm = ops.clip_grad_norm(grads, bound, dtype=to)
            assert abs(norm.item() - want) <= 1.001 * E * want
            for o, g, c in zip(outs, grads, before):
                assert torch.equal(g, c) and o.shape == g.shape and o.dtype == (to or g.dtype)
                exact = g.double().cpu() * factor
                assert_within(o, exact, exact.abs() * (half_step(o.dtype) + 2 * E)
                              + torch.finfo(o.dtype).tiny, "clipped")
                if factor == 1.0 and o.dtype == g.dtype:
                    assert torch.equal(o, g)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_clip_in_place(device, dtype, kind):
    grads = [g for g in gradients(kind, device, dtype) if g.numel() < 2 or 0 not in g.stride()]
    want = norm_of(grads)
    before = [g.clone() for g in grads]
    assert abs(ops.clip_grad_norm_(grads, 2 * want).item() - want) <= 1.001 * E * want
    assert all(torch.equal(a, c) for a, c in zip(grads, before))
    version = grads[0]._version
    ops.clip_grad_norm_(grads, want / 2)
    assert grads[0]._version > version
    for g, c in zip(grads, before):
        exact = c.double().cpu() / 2
        assert_within(g, exact, exact.abs() * (half_step(g.dtype) + 2 * E)
                      + torch.finfo(g.dtype).tiny, "clipped")


@pytest.mark.parametrize("device", BOTH)
def test_clip_leaves_what_lies_between(device):
    flat = torch.ones(100, device=device)
    ops.clip_grad_norm_([flat[3:10], flat[11:50], flat[60:99:2]], 0.0)
    zero = [i for i in range(100) if 3 <= i < 10 or 11 <= i < 50 or (60 <= i < 99 and i % 2 == 0)]
    assert not flat[zero].any() and flat.sum() == 100 - len(zero)


@pytest.mark.parametrize("device", BOTH)
def test_norm_of_extremes(device):
    """Squares outside the range of 32 bits, none and not finite values."""
    t = lambda *x, dtype=torch.float32: torch.tensor(x, dtype=dtype, device=device)  # noqa: E731
    for x in ((3e30, 4e30), (3e-30, 4e-30)):
        assert abs(ops.grad_norm([t(*x)]).item() / (5 / 3 * x[0]) - 1) <= 4 * E
        (y,), _ = ops.clip_grad_norm([t(*x)], x[0] / 1000)
        assert torch.allclose(y / x[0], t(0.6e-3, 0.8e-3), rtol=8 * E, atol=0)
    assert ops.grad_norm([t(3e38, 3e38)]).isinf()
    (y,), n = ops.clip_grad_norm([t(3e38, 3e38)], 1.0)
    assert n.isinf() and torch.allclose(y, t(0.5 ** 0.5, 0.5 ** 0.5), rtol=4 * E, atol=0)
    assert ops.grad_norm(t()).item() == 0.0 and ops.grad_norm([t(0.0), t()]).item() == 0.0
    (y,), n = ops.clip_grad_norm([t(0.0, 0.0)], 0.0)
    assert not y.any() and n == 0
    (y,), n = ops.clip_grad_norm([t()], 1.0)
    assert y.numel() == 0 and n == 0
    (y, z), n = ops.clip_grad_norm([t(1.0, math.inf), t(2.0)], 1.0)
    assert n.isinf() and y[0] == 0 and y[1].isnan() and z == 0
    (y,), n = ops.clip_grad_norm([t(1.0, math.nan)], 1.0)
    assert n.isnan() and y.isnan().all()
    (y,), n = ops.clip_grad_norm([t(1.0, math.inf)], math.inf)
    assert n.isinf() and y[0] == 1 and y[1].isinf()


@pytest.mark.parametrize("device", BOTH)
def test_clip_refuses(device):
    x, y = torch.ones(8, device=device), torch.ones(8, device=device)
    for call in (lambda: ops.grad_norm([]), lambda: ops.grad_norm([x.double()]),
                 lambda: ops.grad_norm([x.int()]), lambda: ops.grad_norm([x.to_sparse()]),
                 lambda: ops.clip_grad_norm([x], -1.0), lambda: ops.clip_grad_norm([x], math.nan),
                 lambda: ops.clip_grad_norm([x, y], 1.0, out=[x]),
                 lambda: ops.clip_grad_norm([x], 1.0, out=[y[:7]]),
                 lambda: ops.clip_grad_norm([x], 1.0, out=[y.double()]),
                 lambda: ops.clip_grad_norm([x], 1.0, out=[y], dtype=torch.float16),
                 lambda: ops.clip_grad_norm([x], 1.0, dtype=torch.int32),
                 lambda: ops.clip_grad_norm([x.new_ones(4, 8)], 1.0, out=[y.expand(4, 8)]),
                 lambda: ops.clip_grad_norm_([x.expand(4, 8)], 1.0),
                 lambda: ops.clip_grad_norm_([x, x], 1.0),
                 lambda: ops.clip_grad_norm_([x[:5], x[4:]], 1.0),
                 lambda: ops.clip_grad_norm([x[:4], y[:4]], 1.0, out=[y[4:], y[2:6]]),
                 lambda: ops.clip_grad_norm([x[:4], x[4:]], 1.0, out=[x[4:], y[:4]])):
        with pytest.raises(ValueError):
            call()
    assert x.sum() == 8 and y.sum() == 8


@pytest.mark.gpu
def test_clip_refuses_two_devices():
    with pytest.raises(ValueError):
        ops.grad_norm([torch.ones(3, device="cuda"), torch.ones(3)])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([torch.ones(3, device="cuda")], 1.0, out=[torch.ones(3)])


@pytest.mark.gpu
def test_clip_repeats_and_replays():
    grads = gradients("many", "cuda", torch.float32) + [torch.randn(3_000_001, device="cuda")]
    out = [torch.empty_like(g) for g in grads]
    ops.clip_grad_norm(grads, 1.0, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = ops.clip_grad_norm(grads, 1.0, out=out)
        alone = ops.grad_norm(grads)
    for factor in (1.0, 3.0, 0.1):
        for g in grads:
            g.mul_(factor)
        graph.replay()
        torch.cuda.synchronize()
        first = [o.clone() for o in out]
        eager, n = ops.clip_grad_norm(grads, 1.0)
        assert torch.equal(n, norm) and torch.equal(n, alone)
        for a, c in zip(first, eager):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_two_streams_and_a_graph():
    """Calls on two streams at once, and two captured graphs replayed in turn,
    each with its own workspaces, against the same calls one by one."""
    def make(seed):
        q, k, v, dout = attention_inputs(2, 150, 150, 4, 2, 64, torch.float16, "cuda", seed)
        grads = [torch.randn(n, device="cuda") for n in (70_001, 33)]
        return [q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True)], dout, grads

    documents = DOCS["packed"](2, 150).cuda()
    positions, frequencies = torch.arange(150, device="cuda"), ops.rotary_frequencies(
        64, device="cuda")

    def work(x):
        leaves, dout, grads = x
        q, k = ops.rotary(*leaves[:2], positions, frequencies, interleaved=True)
        out = ops.attention(q, k, leaves[2], documents)
        clipped, norm = ops.clip_grad_norm(grads, 0.5)
        few = ops.attention(q[:, -1:].detach(), k.detach(), leaves[2].detach(), documents)
        # no graph of the leaves outlives the call: see the test below
        return [out.detach(), few, *torch.autograd.grad(out, leaves, dout), *clipped, norm]

    inputs = [make(1), make(2)]
    want = [work(x) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n] = work(inputs[n])
    torch.cuda.synchronize()
    for a, c in zip(got[0] + got[1], want[0] + want[1]):
        assert torch.equal(a, c)
    graphs, held = [], []
    for x in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(work(x))
    for turn in (0, 1, 0, 0, 1):
        graphs[turn].replay()
        torch.cuda.synchronize()
        for a, c in zip(held[turn], want[turn]):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_captured_backward_beside_an_eager_graph_is_refused():
    """The leaves' gradients would go to another stream than the captured one."""
    q, k, v, dout = attention_inputs(1, 40, 40, 2, 2, 32, torch.float32, "cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    positions, frequencies = torch.arange(40, device="cuda"), ops.rotary_frequencies(
        32, device="cuda")
    calls = (lambda: ops.attention(*leaves),
             lambda: ops.rotary(q, k, positions, frequencies)[0])
    for call in calls:
        alive = call()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(call(), leaves[:1], dout)
        torch.cuda.synchronize()
        torch.autograd.grad(alive, leaves[:1], dout)
