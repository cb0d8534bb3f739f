"""Language-model operators where their callers leave the common path: other
modes of differentiation and tracing, extreme and not finite values, rows of
zeros, block shapes of large inputs.  Oracles and tolerances are those of
test_language_ops.py where nothing else is said."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from deepreduce_amd import ops
from test_language_ops import (BOTH, DOCS, E, TYPES, assert_within, attention_inputs,
                               attention_oracle, check_attention, half_step, pack, seen_pairs)


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


# --------------------------------------------------------------------------
# gradients of all sizes in 16 bits
# --------------------------------------------------------------------------

def relative_error(got, want):
    return ((got.detach().double().cpu() - want).norm() / want.norm()).item()


# P, dS and the result are rounded to half a step each; the errors of thousands
# of pairs are independent, so that they add up as the sums themselves do
THREE_ROUNDINGS = 3 * half_step(torch.float16)


def small_gradient(name, sizes, documents=None):
    """The gradient of leaf `name`, fp16, and its value in 64 bits: one head
    with dout of `sizes`, one for each query, and the leaf itself so small that
    its gradient, with a scale that makes up for it, is not."""
    n = len(sizes)
    x = dict(zip(("q", "k", "v", "dout"),
                 attention_inputs(1, n, n, 1, 1, 64, torch.float32, "cuda")))
    x["dout"] = x["dout"] * sizes.cuda().view(1, n, 1, 1)
    x[name] = x[name] * 2.0 ** -16
    q, k, v, dout = (t.half() for t in x.values())
    leaves = {"q": q.requires_grad_(True), "k": k.requires_grad_(True)}
    out = ops.attention(q, k, v, documents=documents, scale=2.0 ** 13)
    (got,) = torch.autograd.grad(out, leaves[name], dout)
    return got, attention_oracle(q, k, v, documents, None, False, 2.0 ** 13, dout)["d" + name][0]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["q", "k"])
@pytest.mark.parametrize("zeros", ["front", "between", "none"])
def test_queries_without_a_gradient_cost_no_bits(name, zeros):
    """Small gradients beside queries that have none, such as unscored tokens."""
    sizes = torch.full((4096,), 3e-7)
    if zeros == "front":
        sizes[:64] = 0
    if zeros == "between":
        sizes.view(-1, 256)[:, 100:200] = 0
    assert relative_error(*small_gradient(name, sizes)) <= THREE_ROUNDINGS


@pytest.mark.gpu
def test_gradients_of_other_sizes():
    """A document whose gradients are 300000 times those of the next, which begins
    inside a tile; and queries of both sizes in turn."""
    n, edge, tile = 2400, 200, 256
    sizes = torch.full((n,), 3e-7)
    sizes[:edge], sizes[edge:tile] = 0.1, 0
    documents = torch.tensor([pack([edge, n - edge], n)], dtype=torch.int32, device="cuda")
    got, want = small_gradient("k", sizes, documents)
    assert relative_error(got[:, :edge], want[:, :edge]) <= THREE_ROUNDINGS
    assert relative_error(got[:, edge:], want[:, edge:]) <= THREE_ROUNDINGS
    sizes = torch.full((n,), 3e-7)
    sizes[::2] = 0.1
    got, want = small_gradient("q", sizes)
    assert relative_error(got[:, ::2], want[:, ::2]) <= THREE_ROUNDINGS
    assert relative_error(got[:, 1::2], want[:, 1::2]) <= THREE_ROUNDINGS


# --------------------------------------------------------------------------
# clipping
# --------------------------------------------------------------------------

@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("to", TYPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("count,bound", [(100, 1e-3), (100, 1e-6), (40_001, 1e-5), (3, 1e30)])
def test_clip_of_exploding_gradients(device, dtype, to, count, bound):
    """Factors that 32 bits hold as subnormal numbers or not at all."""
    gen = torch.Generator().manual_seed(count)
    x = (3e38 * (0.5 + 0.5 * torch.rand(count, generator=gen))).to(dtype)
    norm = math.sqrt(math.fsum((x.double() ** 2).tolist()))
    (y,), n = ops.clip_grad_norm([x.to(device)], bound, dtype=to)
    assert n.isinf() == (norm > torch.finfo(torch.float32).max)
    want = x.double() * (bound / norm)
    if bound > torch.finfo(to).max:
        assert y.isinf().all()
        return
    # rounded to 32 bits and to the type; below its normal numbers a fixed half step
    info = torch.finfo(to)
    least = info.tiny * info.eps / 2
    assert_within(y, want, want.abs() * (half_step(to) + 2 * E) + least * 1.001, "clipped")


# --------------------------------------------------------------------------
# many requests
# --------------------------------------------------------------------------

def time_of(call):
    """Seconds of a call among others, the least of three groups."""
    for _ in range(3):
        call()
    least = math.inf
    for _ in range(3):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(5):
            call()
        end.record()
        torch.cuda.synchronize()
        least = min(least, begin.elapsed_time(end) / 5e3)
    return least


@pytest.mark.gpu
def test_many_requests_read_their_keys_once():
    """Heads that share keys read them together at any number of requests: well
    within the time of a few copies (once a query head takes 20 copies)."""
    q = torch.randn(32, 1, 16, 64, device="cuda")
    k, v = (torch.randn(32, 32768, 1, 64, device="cuda") for _ in range(2))
    copies = time_of(lambda: (k.clone(), v.clone()))
    assert time_of(lambda: ops.attention(q, k, v)) <= 4 * copies


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(64, 1, 700, 12, 4, 64), (40, 2, 601, 16, 1, 128),
                                   (600, 1, 300, 3, 1, 32), (33, 5, 1111, 16, 2, 40)], ids=str)
def test_many_requests(dtype, shape):
    b, sq, sk, hq, hkv, d = shape
    q, k, v, dout = attention_inputs(*shape, dtype, "cuda", seed=sum(shape))
    lengths = torch.randint(0, sk, (b,), generator=torch.Generator().manual_seed(b))
    documents = torch.tensor([pack([n], sk) for n in lengths], dtype=torch.int32)
    documents[::3] = 4  # whole caches, and padding behind the others
    slopes = torch.linspace(0.05, 0.0, hq, device="cuda")
    check_attention(q, k, v, dout, documents.cuda(), slopes, causal=True)
    check_attention(q, k, v, dout, causal=sq > 1)


# --------------------------------------------------------------------------
# steps that are not finite
# --------------------------------------------------------------------------

def spoil(x, which, bad, where):
    """Copies of x's tensors with `bad` in one value of `which`, or in all."""
    y = {n: t.clone() for n, t in x.items()}
    t = y[which]
    if where == "all":
        t[:] = bad
    else:
        t[0, t.shape[1] * 2 // 3, t.shape[2] - 1, 5] = bad
    return y


def attention_step(x, **options):
    leaves = [x[n].detach().requires_grad_(True) for n in ("q", "k", "v")]
    out = ops.attention(*leaves, **options)
    return [out.detach(), *torch.autograd.grad(out, leaves, x["dout"])]


def formulas(q, k, v, dout, documents, causal):
    """Results of one entry in 64 bits; hidden pairs are in no product."""
    sq, hq, d = q.shape
    sk, hkv = k.shape[:2]
    seen, _ = seen_pairs(documents.unsqueeze(0), causal, 1, sq, sk)
    seen = seen[0]

    def product(w, x, s):
        bad = ~x.isfinite()
        y = w @ x.masked_fill(bad, 0.0)
        for j in bad.any(1).nonzero().flatten().tolist():
            y = y + torch.where(s[:, j:j + 1], w[:, j:j + 1] * x[j].masked_fill(~bad[j], 0.0), 0.0)
        return y

    got = {n: torch.zeros(t.shape, dtype=torch.float64)
           for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    for h in range(hq):
        g, scale = h * hkv // hq, d ** -0.5
        Q, K, V, dO = q[:, h], k[:, g], v[:, g], dout[:, h]
        s = (scale * (Q @ K.T)).masked_fill(~seen, -math.inf)
        P = torch.where(seen, torch.softmax(s, 1), 0.0)
        O = product(P, V, seen)
        dP = torch.where(seen, dO @ V.T, 0.0)
        delta = torch.where(seen.any(1), (dO * O).sum(1), 0.0).unsqueeze(1)
        dS = torch.where(seen, P * (dP - delta), 0.0)
        got["out"][:, h], got["dq"][:, h] = O, scale * product(dS, K, seen)
        got["dk"][:, g] += scale * product(dS.T, Q, seen.T)
        got["dv"][:, g] += product(P.T, dO, seen.T)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [math.inf, math.nan], ids=str)
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("where", ["one", "all"])
@pytest.mark.parametrize("shape", [(1, 300, 300, 2, 1, 64), (1, 100, 333, 2, 2, 40),
                                   (1, 3, 1000, 4, 2, 128), (32, 130, 130, 16, 16, 32)], ids=str)
def test_what_is_not_finite_stays_where_it_is_seen(dtype, bad, which, where, shape):
    """What a row sees that is not finite makes it so, as in the formulas; rows that
    do not see it are those of a call without it, and hidden NaN change nothing."""
    b, sq, sk, hq, hkv, d = shape
    names = ("q", "k", "v", "dout")
    x = dict(zip(names, attention_inputs(*shape, dtype, "cpu", seed=sk)))
    n = sk - sk // 4
    documents = torch.tensor([pack([n - 7, 7], n)] * b, dtype=torch.int32)
    documents = torch.cat((documents, torch.full((b, sk - n), 2, dtype=torch.int32)), 1)
    dirty = spoil(x, which, bad, where)
    hidden = {n: t.clone() for n, t in dirty.items()}
    for t in hidden.values():  # the last document, which no check below looks at
        t[:, -(sk // 4):] = math.nan
    for causal in (False, True):
        on = lambda y, e=slice(None): {n: t[e].cuda() for n, t in y.items()}  # noqa: E731
        options = dict(documents=documents.cuda(), causal=causal)
        got = attention_step(on(dirty), **options)
        more = attention_step(on(hidden), **options)
        clean = attention_step(on(x), **options)
        want = formulas(*[dirty[n][0].double() for n in names], documents[0], causal)
        for name, g, m, c in zip(("out", "dq", "dk", "dv"), got, more, clean):
            g, m, c, w = (t.double().cpu() for t in (g, m, c, want[name].unsqueeze(0)))
            assert torch.equal(g[:1].isfinite(), w.isfinite()), name
            seen = slice(0, max(0, g.shape[1] - sk // 4))
            assert torch.equal(g[:, seen].isfinite(), m[:, seen].isfinite()), name
            fine = g.isfinite()
            size = c.abs().max()
            # scores and sums as in a clean call, or added in another order
            tol = 8 * (half_step(dtype) + 256 * E) * size
            fine[0] &= False
            if where == "one":
                assert ((g - c).abs()[fine] <= tol).all() and fine[1:].all(), name
            both = g[:1].isfinite()
            assert ((g[:1] - w).abs()[both] <= 2 * tol).all(), name
            both = g[:, seen].isfinite()
            assert ((g[:, seen] - m[:, seen]).abs()[both] <= tol).all(), name


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sq", [1, 70])
def test_scores_of_minus_infinity(device, dtype, sq):
    """A query whose scores are all minus infinity sees nothing: it gives 0, with
    zero gradients."""
    q, k, v, dout = attention_inputs(1, sq, 70, 2, 2, 32, dtype, device)
    q[..., 3] = q[..., 3].abs() + 1
    k[..., 3] = -math.inf
    x = dict(q=q, k=k, v=v, dout=dout)
    for causal in (False, True):
        for t in attention_step(x, causal=causal):
            assert not t.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("which,bad,where", [
    ("v", math.nan, "all"), ("q", math.nan, "all"), ("dout", math.nan, "all"),
    ("dout", math.inf, "all"), ("dout", math.inf, "one"), ("dout", math.nan, "one"),
    ("v", math.inf, "one"), ("v", math.nan, "one"), ("k", math.inf, "one"),
    ("q", math.inf, "one")])
def test_steps_that_are_not_finite(dtype, which, bad, where):
    """Overflow is an ordinary step under loss scaling: one that is NaN all over
    takes no longer than others, and one value that is not finite makes no more
    rows be done again than share a tile with it (all of them: 100 to 800 times)."""
    x = dict(zip(("q", "k", "v", "dout"),
                 attention_inputs(1, 2048, 2048, 4, 4, 64, dtype, "cuda")))
    dirty = spoil(x, which, bad, where)
    documents = torch.zeros(1, 2048, dtype=torch.int32, device="cuda")
    documents[:, :900] = 1
    for options in (dict(causal=True), dict(documents=documents)):
        usual = time_of(lambda: attention_step(x, **options))
        this = time_of(lambda: attention_step(dirty, **options))
        print(f"\n{this * 1e6:.0f} us, usual {usual * 1e6:.0f}", end="")
        assert this <= (2 if where == "all" and bad != math.inf else 64) * usual


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_caches_of_anything_behind_their_sequences(dtype):
    """Tokens over caches whose padding holds NaN, in time and results those of
    caches that hold zeros there."""
    b, sk = 8, 8192
    q, k, v, _ = attention_inputs(b, 1, sk, 12, 4, 64, dtype, "cuda")
    lengths = [8191, 5000, 4097, 4095, 33, 1, 7000, 6432]
    ahead = torch.tensor([pack([n], sk - 1) + [0] for n in lengths], dtype=torch.int32,
                         device="cuda")
    behind = torch.tensor([[-1] * (sk - n) + [0] * n for n in lengths], dtype=torch.int32,
                          device="cuda")
    for documents in (ahead, behind):
        hidden = (documents < 0)[..., None, None]
        zeros, anything = ([t.masked_fill(hidden, x) for t in (k, v)] for x in (0.0, math.nan))
        want = ops.attention(q, *zeros, documents)
        assert want.isfinite().all()
        assert torch.equal(ops.attention(q, *anything, documents), want)
        usual = time_of(lambda: ops.attention(q, *zeros, documents))
        this = time_of(lambda: ops.attention(q, *anything, documents))
        print(f"\n{this * 1e6:.0f} us, usual {usual * 1e6:.0f}", end="")
        assert this <= 2 * usual


# --------------------------------------------------------------------------
# views that torch negates when it reads them
# --------------------------------------------------------------------------

def negated(x):
    """A view with x's values over memory that holds their negatives."""
    view = torch._neg_view(-x)
    assert view.is_neg() and torch.equal(view, x)
    return view


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("name", ["attention", "rotary", "grad_norm", "clip_grad_norm"])
def test_negated_views(device, name):
    call, inputs = small_calls(device)[name]
    want = call(*inputs)
    for n, x in enumerate(inputs):
        others = list(inputs)
        others[n] = negated(x)
        assert torch.equal(call(*others), want)
    assert torch.equal(call(*[negated(x) for x in inputs]), want)


@pytest.mark.parametrize("device", BOTH)
def test_negated_gradients(device):
    q, k, v, dout = attention_inputs(1, 9, 9, 2, 1, 16, torch.float32, device)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    positions = torch.arange(9, device=device)
    frequencies = ops.rotary_frequencies(16, device=device)
    for call in (lambda: ops.attention(q, k, v), lambda: ops.rotary(q, k, positions,
                                                                     frequencies)[0]):
        want, got = (torch.autograd.grad(call(), leaves[:1], g) for g in (dout, negated(dout)))
        assert torch.equal(want[0], got[0])
    x, y = (torch.randn(40, device=device) for _ in range(2))
    (want,), _ = ops.clip_grad_norm([x], 0.5)
    for out in (torch.empty_like(x), negated(y)):
        ops.clip_grad_norm([x], 0.5, out=[out])
        assert torch.equal(out, want)
    view = negated(x)
    ops.clip_grad_norm_([view], 0.5)
    assert torch.equal(view, want)


# --------------------------------------------------------------------------
# the blocks of large inputs
# --------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [
    (32, 129, 129, 16, 16, 64),   # a last block with one row; 1024 blocks
    (16, 200, 200, 16, 16, 32),   # 512 blocks: long and short ones alternate
    (24, 161, 161, 12, 12, 128), (40, 140, 140, 16, 8, 96),
    (64, 130, 197, 8, 8, 40),     # queries behind 67 keys
    (600, 33, 33, 1, 1, 64)], ids=str)
@pytest.mark.parametrize("docs", ["none", "packed", "mixed"])
def test_large_batches(dtype, shape, docs):
    """Rows enough for blocks of four waves that share their tiles, in all
    kernels: some entries against 64 bits, the others against the same entry
    alone, which takes other blocks."""
    b, sq, sk, hq, hkv, d = shape
    assert b * hkv * ((min(sq, sk) + 127) // 128) >= 512
    x = attention_inputs(*shape, dtype, "cuda", seed=sum(shape))
    documents = DOCS[docs](b, sk)
    documents = None if documents is None else documents.cuda()
    for causal in (False, True):
        slopes = torch.linspace(0.3, 0.0, hq).cuda() if causal else None
        run = lambda e: attention_step(  # noqa: E731
            {n: t[e] for n, t in zip(("q", "k", "v", "dout"), x)}, slopes=slopes, causal=causal,
            documents=None if documents is None else documents[e])
        got = run(slice(None))
        for e in range(b):
            one = slice(e, e + 1)
            if e in (0, b // 2, b - 1):
                want = attention_oracle(*[t[one] for t in x[:3]],
                                        None if documents is None else documents[one], slopes,
                                        causal, d ** -0.5, x[3][one])
                for name, g in zip(("out", "dq", "dk", "dv"), got):
                    assert_within(g[one], *want[name], f"{name} of entry {e}")
            elif e % max(1, b // 20) == 0:
                for name, g, w in zip(("out", "dq", "dk", "dv"), got, run(one)):
                    # both off by their roundings: of P or dS, and of the result
                    tol = 4 * (half_step(dtype) + 256 * E) * w.abs().max()
                    assert (g[one].double() - w.double()).abs().max() <= tol, f"{name} of {e}"


# --------------------------------------------------------------------------
# scores beyond what 32 bits hold to 1
# --------------------------------------------------------------------------

@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", ["large", "one", "negative"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 8), (2, 70, 70, 4, 2, 64),
                                   (1, 2, 900, 4, 1, 128), (1, 300, 333, 2, 2, 40)], ids=str)
def test_far_scores(device, dtype, size, shape):
    """The one key of the largest score has all of the probability, in every row
    or in those of one query and one key whose values are large."""
    b, sq, sk, hq, hkv, d = shape
    q, k, v, dout = attention_inputs(*shape, dtype, "cpu", seed=sum(shape))
    if size == "one":
        q[:, sq // 2] *= 8e3
        k[:, sk // 3] *= 8e3
    else:
        q, k = q.abs() * 6000, k.abs() * 6000
        if size == "negative":
            k = -k
    documents = torch.tensor([pack([sk // 2, sk - sk // 2 - 1], sk)] * b, dtype=torch.int32)
    documents[:, -1] = 5
    for causal in (False, True):
        got = attention_step({n: t.to(device) for n, t in
                              dict(q=q, k=k, v=v, dout=dout).items()},
                             documents=documents.to(device), causal=causal)
        for e in range(b):
            want = formulas(*[t[e].double() for t in (q, k, v, dout)], documents[e], causal)
            far = torch.zeros(hq, sq, dtype=torch.bool)
            seen, _ = seen_pairs(documents[e:e + 1], causal, 1, sq, sk)
            for h in range(hq):
                s = d ** -0.5 * (q[e, :, h].double() @ k[e, :, h * hkv // hq].double().T)
                top = s.masked_fill(~seen[0], -math.inf).amax(1)
                s2 = s.masked_fill(~seen[0], -math.inf).topk(min(2, sk), 1).values
                # rows whose two largest scores differ by more than their own
                # roundings: d products, their sums and the scaling in 32 bits
                size_of = d ** -0.5 * (q[e, :, h].double().abs()
                                       @ k[e, :, h * hkv // hq].double().abs().T)
                off = (d + 4) * E * torch.where(seen[0], size_of, 0.0).amax(1)
                far[h] = (s2[:, 0] - s2[:, -1] > 2 * off + 200) | (seen[0].sum(1) == 1)
                far[h] &= top.isfinite()
            assert far.any() and (size == "one" or far.float().mean() > 0.2)
            # those rows are one value of V, rounded nowhere
            rows = far.T
            tol = 1.01 * half_step(dtype) * want["out"].abs() + 1e-6
            assert ((got[0][e].double().cpu() - want["out"]).abs() <= tol)[rows].all()
            if size != "one" and far.all():
                sums = (sq * hq // hkv + 4) * E
                for n, name in ((1, "dq"), (2, "dk"), (3, "dv")):
                    g, w = got[n][e].double().cpu(), want[name]
                    least = 1e-6 * (1 + w.abs().max())
                    if name != "dv":  # differences of equal products
                        least = 1e-4 * d ** -0.5 * max(q.abs().max(), k.abs().max()).item()
                    assert ((g - w).abs() <= (half_step(dtype) + sums) * w.abs() + least).all(), name
