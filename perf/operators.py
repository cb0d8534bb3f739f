"""The framework's language-model operators as measurable cases: attention over
packed documents, rotary positions, the global gradient norm and clipping.

`run` computes each operator in a plain form (elementary torch operations in
32 bits, rounded once) or, where `own` is true, calls `deepreduce_amd.ops`.
`exact` is the same in 64 bits.  Shapes are those of this repository's models
(BERT-base, the LSTM language model, ResNet-20) or generic ones around them.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def listed():
    return [
        # serving: one new token of 8 left-padded requests over a long cache
        # with 3 query heads on each key-value head
        dict(name="attn_token_bf16", op="attention", train=False, b=8, sq=1, sk=32768,
             hq=12, hkv=4, d=64, type="bf16", docs="left", mean=0, layout=1,
             slopes=False, causal=True),
        # training BERT on packed rows: the encoder's 512 positions hold
        # several documents and some padding
        dict(name="attn_packed_train_bf16", op="attention", train=True, b=32, sq=512,
             sk=512, hq=12, hkv=12, d=64, type="bf16", docs="packed", mean=160, layout=2,
             slopes=False, causal=False),
        # training without autocast at an odd length, distance bias in place
        # of learned positions
        dict(name="attn_ragged_train_fp32", op="attention", train=True, b=3, sq=333,
             sk=333, hq=12, hkv=12, d=64, type="fp32", docs="packed", mean=90, layout=3,
             slopes=True, causal=False),
        # training a decoder on long rows, heads of 128 shared by four
        dict(name="attn_causal_train_fp16", op="attention", train=True, b=2, sq=4096,
             sk=4096, hq=16, hkv=4, d=128, type="fp16", docs="none", mean=0, layout=4,
             slopes=True, causal=True),
        # encoding a long row of long documents
        dict(name="attn_long_forward_bf16", op="attention", train=False, b=1, sq=16384,
             sk=16384, hq=12, hkv=12, d=64, type="bf16", docs="packed", mean=5000, layout=5,
             slopes=False, causal=False),
        # serving: one token of 8 requests, far into a long context
        dict(name="rotary_token_fp16", op="rotary", train=False, b=8, s=1, hq=12, hkv=4,
             d=64, dim=64, interleaved=False, factor=8.0, far=1_000_000, type="fp16"),
        # training BERT's packed rows, forward and back
        dict(name="rotary_train_bf16", op="rotary", train=True, b=32, s=512, hq=12, hkv=12,
             d=64, dim=64, interleaved=False, factor=1.0, far=512, type="bf16"),
        # a long prompt at an odd length, half of each head rotated, neighbours paired
        dict(name="rotary_long_fp32", op="rotary", train=False, b=2, s=8191, hq=16, hkv=4,
             d=128, dim=64, interleaved=True, factor=4.0, far=131_072, type="fp32"),
        # monitoring the LSTM language model's gradients
        dict(name="norm_rnn_fp32", op="norm", shapes="rnn", type="fp32", flat=False, layout=1),
        # a large model's gradients in buckets at odd offsets, two types
        dict(name="norm_mixed_bf16", op="norm", shapes="mixed", type="bf16", flat=True, layout=2,
             count=120, top=27, most=1 << 28),
        # clipping ResNet-20: 65 small tensors, where latency counts
        dict(name="clip_resnet20_fp32", op="clip", shapes="resnet20", type="fp32", flat=False,
             layout=3, max_norm=1.0),
        # clipping BERT-base between backward and the exchange
        dict(name="clip_bert_fp32", op="clip", shapes="bert", type="fp32", flat=False, layout=4,
             max_norm=1.0),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotary", "norm", "clip"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    layout = rng.randrange(10, 1 << 30)
    if op == "attention":
        use = rng.choice(["token", "train", "train", "forward"])
        d = rng.choice([32, 40, 64, 64, 80, 96, 128])
        hkv = rng.choice([1, 2, 3, 4, 6])
        hq = hkv * rng.choice([1, 1, 2, 3, 4])
        if use == "token":
            sk = _spread(rng, 1, 32768)
            sq = min(sk, rng.choice([1, 1, 2, 5]))
            b = _spread(rng, 1, max(1, min(32, (1 << 26) // (sk * hkv * d))))
            docs, causal = rng.choice(["left", "none"]), True
        else:
            # no more pairs than the largest listed cases have
            most = 16 * 128 * 4096 ** 2 * (1 if use == "train" else 3)
            if kind == "fp32":
                most //= 16
            most //= hq * d
            sq = sk = _spread(rng, 16, min(16384, math.isqrt(most)))
            b = _spread(rng, 1, max(1, min(32, most // (sk * sk))))
            docs, causal = rng.choice(["packed", "packed", "none"]), rng.random() < 0.4
        return dict(op="attention", train=use == "train", b=b, sq=sq, sk=sk, hq=hq, hkv=hkv,
                    d=d, type=kind, docs=docs, mean=_spread(rng, 1, sk), layout=layout,
                    slopes=rng.random() < 0.4, causal=causal)
    if op == "rotary":
        d = rng.choice([32, 40, 64, 80, 96, 128])
        s = _spread(rng, 1, 8192)
        hkv = rng.choice([1, 2, 3, 4, 12])
        return dict(op="rotary", train=rng.random() < 0.5,
                    b=_spread(rng, 1, max(1, min(64, 16384 // s))), s=s,
                    hq=hkv * rng.choice([1, 2, 3]), hkv=hkv, d=d,
                    dim=rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]),
                    interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 2.0, 8.0]),
                    far=_spread(rng, s, 1_000_000) if s > 1 else _spread(rng, 2, 1_000_000),
                    type=kind)
    case = dict(op=op, shapes="mixed", type=kind, flat=rng.random() < 0.5, layout=layout,
                count=_spread(rng, 1, 400), top=rng.randint(8, 24), most=1 << 26)
    if op == "clip":
        case["max_norm"] = rng.choice([0.01, 1.0, 1e6])
    return case


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _documents(case):
    """Document numbers [b][sk] of a case, -1 for padding; None without them."""
    if case["docs"] == "none":
        return None
    rng = random.Random(case["layout"])
    rows = []
    for _ in range(case["b"]):
        sk = case["sk"]
        if case["docs"] == "left":  # requests of different lengths, padded in front
            pad = rng.randint(0, sk // 2)
            rows.append([-1] * pad + [0] * (sk - pad))
            continue
        row, number = [], 0
        used = sk - (rng.randint(0, sk // 8) if rng.random() < 0.7 else 0)
        while len(row) < used:
            n = min(used - len(row), rng.randint(1, 2 * case["mean"]))
            row += [number] * n
            number += 1
        rows.append(row + [-1] * (sk - used))
    return rows


def _sizes(case):
    """The shapes and types of a case's gradients."""
    if case["shapes"] == "rnn":  # the LSTM language model's parameters
        shapes = [(10_004, 96), (2680, 96), (2680, 670), (2680,), (2680,), (96, 670), (96,),
                  (10_004, 96), (10_004,)]
    elif case["shapes"] == "resnet20":
        shapes = [(16, 3, 3, 3), (16,), (16,)]
        width = 16
        for out in (16, 32, 64):
            for block in range(3):
                shapes += [(out, width, 3, 3), (out,), (out,), (out, out, 3, 3), (out,), (out,)]
                if width != out:
                    shapes += [(out, width, 1, 1), (out,), (out,)]
                width = out
        shapes += [(10, 64), (10,)]
    elif case["shapes"] == "bert":
        h = 768
        shapes = [(30_522, h), (512, h), (h,), (h,)]
        for _ in range(12):
            shapes += [(3 * h, h), (3 * h,), (h, h), (h,), (h,), (h,), (4 * h, h), (4 * h,),
                       (h, 4 * h), (h,), (h,), (h,)]
    else:  # many sizes, odd ones among them, a few in 32 bits
        rng = random.Random(case["layout"])
        shapes, left = [], case["most"]
        for _ in range(case["count"]):
            n = min(_spread(rng, 1, 1 << case["top"]), left)
            left -= n
            if n:
                shapes.append((n,))
        return [(s, "fp32" if rng.random() < 0.2 else case["type"]) for s in shapes]
    return [(s, case["type"]) for s in shapes]


def _normal(gen, shape, kind, sigma=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * sigma).to(_TYPES[kind])


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case.get("type")
    if case["op"] == "attention":
        b, sq, sk, hq, hkv, d = (case[n] for n in ("b", "sq", "sk", "hq", "hkv", "d"))
        x = {"q": _normal(gen, (b, sq, hq, d), kind), "k": _normal(gen, (b, sk, hkv, d), kind),
             "v": _normal(gen, (b, sk, hkv, d), kind)}
        if case["train"]:
            x["do"] = _normal(gen, (b, sq, hq, d), kind)
        rows = _documents(case)
        x["documents"] = None if rows is None else torch.tensor(rows, dtype=torch.int32,
                                                                device="cuda")
        x["slopes"] = None
        if case["slopes"]:  # a geometric row of slopes, as distance biases are set
            x["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)],
                                       device="cuda")
        return x
    if case["op"] == "rotary":
        b, s, d = case["b"], case["s"], case["d"]
        x = {"q": _normal(gen, (b, s, case["hq"], d), kind),
             "k": _normal(gen, (b, s, case["hkv"], d), kind)}
        if case["train"]:
            x["dq"] = _normal(gen, (b, s, case["hq"], d), kind)
            x["dk"] = _normal(gen, (b, s, case["hkv"], d), kind)
        first = torch.randint(0, max(1, case["far"] - s), (b, 1), generator=gen, device="cuda")
        x["positions"] = first + torch.arange(s, device="cuda")
        return x
    parts = _sizes(case)
    if case["flat"]:  # views of one bucket for each type, packed without gaps
        total = {}
        for shape, k in parts:
            total[k] = total.get(k, 1) + math.prod(shape)
        bucket = {k: _normal(gen, (n,), k, 0.01) for k, n in total.items()}
        at, grads = {k: 1 for k in total}, []
        for shape, k in parts:
            n = math.prod(shape)
            grads.append(bucket[k][at[k]:at[k] + n].view(shape))
            at[k] += n
    else:
        grads = [_normal(gen, shape, k, 0.01) for shape, k in parts]
    return {"grads": grads}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=dict(case))
    if case["op"] == "attention" and case["train"] and own:
        for n in ("q", "k", "v"):
            state[n].requires_grad_(True)
    if case["op"] == "rotary":
        state["frequencies"] = _frequencies(case)
        if own:
            from deepreduce_amd import ops

            state["frequencies"] = ops.rotary_frequencies(case["dim"], factor=case["factor"],
                                                          device="cuda")
            if case["train"]:
                state["q"].requires_grad_(True)
                state["k"].requires_grad_(True)
    if case["op"] == "clip":  # into the flat buffers that the exchange compresses from
        state["flat"] = {k: torch.cat([g.flatten() for g in part])
                         for k, part in _by_type(state["grads"])}
        at, state["out"] = {k: 0 for k in state["flat"]}, []
        for g in state["grads"]:
            n = at[g.dtype]
            at[g.dtype] += g.numel()
            state["out"].append(state["flat"][g.dtype][n:at[g.dtype]].view(g.shape))
    return state


def _by_type(grads):
    """[(type, its gradients)] in the order of the first of each type."""
    kinds = list(dict.fromkeys(g.dtype for g in grads))
    return [(k, [g for g in grads if g.dtype == k]) for k in kinds]


# --------------------------------------------------------------------------
# the operators
# --------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return {"attention": _attention, "rotary": _rotary, "norm": _norm, "clip": _clip}[
        case["op"]](state, case)


def _visible(documents, causal, sq, sk, b, device):
    """[sq, sk] truth values of one batch entry, None where all are visible."""
    p = torch.arange(sk - sq, sk, device=device).unsqueeze(1)
    j = torch.arange(sk, device=device).unsqueeze(0)
    seen = None
    if documents is not None:
        row = documents[b]
        seen = (row[sk - sq:].unsqueeze(1) == row.unsqueeze(0)) & (row.unsqueeze(0) >= 0)
    if causal:
        seen = j <= p if seen is None else seen & (j <= p)
    return seen, (p - j).abs()


def _attention(state, case):
    q, k, v = state["q"], state["k"], state["v"]
    documents, slopes = state["documents"], state["slopes"]
    if own:
        from deepreduce_amd import ops

        out = ops.attention(q, k, v, documents=documents, slopes=slopes, causal=case["causal"])
        if not case["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["do"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}

    b, sq, hq, d = q.shape
    sk, hkv = k.shape[1:3]
    group, scale = hq // hkv, d ** -0.5
    got = {"out": torch.empty_like(q)}
    if case["train"]:
        got.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
    for e in range(b):
        seen, far = _visible(documents, case["causal"], sq, sk, e, q.device)
        qf = q[e].float().transpose(0, 1).contiguous()
        kf = k[e].float().transpose(0, 1).repeat_interleave(group, 0).contiguous()
        vf = v[e].float().transpose(0, 1).repeat_interleave(group, 0).contiguous()
        p = torch.matmul(qf, kf.transpose(1, 2).contiguous()) * scale
        if slopes is not None:
            p -= slopes.view(hq, 1, 1) * far
        if seen is not None:
            p = p.masked_fill_(~seen, -math.inf)
        top = p.amax(2, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = p.sub_(top).exp_()
        total = p.sum(2, keepdim=True)
        p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
        o = torch.matmul(p, vf)
        got["out"][e] = o.transpose(0, 1)
        if case["train"]:
            do = state["do"][e].float().transpose(0, 1).contiguous()
            dv = torch.matmul(p.transpose(1, 2).contiguous(), do)
            ds = torch.matmul(do, vf.transpose(1, 2).contiguous())
            ds = ds.sub_((do * o).sum(2, keepdim=True)).mul_(p)
            got["dq"][e] = (torch.matmul(ds, kf) * scale).transpose(0, 1)
            dk = torch.matmul(ds.transpose(1, 2).contiguous(), qf) * scale
            got["dk"][e] = dk.view(hkv, group, sk, d).sum(1).transpose(0, 1)
            got["dv"][e] = dv.view(hkv, group, sk, d).sum(1).transpose(0, 1)
    return got


def _frequencies(case):
    i = torch.arange(0, case["dim"], 2, dtype=torch.float64, device="cuda")
    return 10000.0 ** (-i / case["dim"]) / case["factor"]


def _turn(x, cos, sin, case):
    """Rotates the first `dim` values of each head by the angles of [b, s, dim / 2]."""
    n = case["dim"]
    y = x.float()
    if case["interleaved"]:
        a, c = y[..., 0:n:2], y[..., 1:n:2]
        turned = torch.stack((a * cos - c * sin, a * sin + c * cos), -1).flatten(-2)
    else:
        a, c = y[..., :n // 2], y[..., n // 2:n]
        turned = torch.cat((a * cos - c * sin, a * sin + c * cos), -1)
    return torch.cat((turned, y[..., n:]), -1).to(x.dtype)


def _rotary(state, case):
    q, k = state["q"], state["k"]
    if own:
        from deepreduce_amd import ops

        yq, yk = ops.rotary(q, k, state["positions"], state["frequencies"],
                            interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": yq, "k": yk}
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (state["dq"], state["dk"]))
        return {"q": yq.detach(), "k": yk.detach(), "dq": dq, "dk": dk}
    # angles of far positions need 64 bits
    angle = state["positions"].double().unsqueeze(-1) * state["frequencies"]
    cos, sin = angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)
    got = {"q": _turn(q, cos, sin, case), "k": _turn(k, cos, sin, case)}
    if case["train"]:
        got["dq"] = _turn(state["dq"], cos, -sin, case)
        got["dk"] = _turn(state["dk"], cos, -sin, case)
    return got


def _plain_norm(grads):
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _norm(state, case):
    if own:
        from deepreduce_amd import ops

        return {"norm": ops.grad_norm(state["grads"])}
    return {"norm": _plain_norm(state["grads"])}


def _clip(state, case):
    if own:
        from deepreduce_amd import ops

        _, norm = ops.clip_grad_norm(state["grads"], case["max_norm"], out=state["out"])
        return {"norm": norm, "out": list(state["flat"].values())}
    norm = _plain_norm(state["grads"])
    factor = torch.where(norm <= case["max_norm"], torch.ones_like(norm), case["max_norm"] / norm)
    for o, g in zip(state["out"], state["grads"]):
        o.copy_(g.float() * factor)
    return {"norm": norm, "out": list(state["flat"].values())}


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, x)
    if case["op"] == "rotary":
        # each pair is a complex number times exp(i t)
        angle = x["positions"].double()[..., None, None] * _frequencies(case)
        turn = torch.polar(torch.ones_like(angle), angle)

        def turned(t, by):
            y = t.double().clone()
            n = case["dim"]
            even, odd = ((slice(0, n, 2), slice(1, n, 2)) if case["interleaved"]
                         else (slice(0, n // 2), slice(n // 2, n)))
            z = torch.complex(y[..., even].contiguous(), y[..., odd].contiguous()) * by
            y[..., even], y[..., odd] = z.real, z.imag
            return y

        got = {"q": turned(x["q"], turn), "k": turned(x["k"], turn)}
        if case["train"]:
            got["dq"], got["dk"] = turned(x["dq"], turn.conj()), turned(x["dk"], turn.conj())
        return got
    norm = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in x["grads"]))
    if case["op"] == "norm":
        return {"norm": torch.tensor(norm, dtype=torch.float64)}
    factor = min(1.0, case["max_norm"] / norm) if norm else 1.0
    return {"norm": torch.tensor(norm, dtype=torch.float64),
            "out": [torch.cat([g.double().flatten() * factor for g in part])
                    for _, part in _by_type(x["grads"])]}


def _exact_attention(case, x):
    b, sq, sk, hq, hkv, d = (case[n] for n in ("b", "sq", "sk", "hq", "hkv", "d"))
    names = {"out": (x["q"], hq)}
    if case["train"]:
        names.update(dq=(x["q"], hq), dk=(x["k"], hkv), dv=(x["v"], hkv))
    got = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
           for n, (t, _) in names.items()}
    at = torch.arange(sk, device="cuda")
    for e in range(b):
        hidden = torch.zeros(sq, sk, dtype=torch.bool, device="cuda")
        if x["documents"] is not None:
            key = x["documents"][e].long()
            hidden |= key[sk - sq:, None] != key[None, :]
            hidden |= (key < 0)[None, :]
        if case["causal"]:
            hidden |= at[None, :] > at[sk - sq:, None]
        empty = hidden.all(1)
        for h in range(hq):
            g = h // (hq // hkv)
            q, k, v = x["q"][e, :, h].double(), x["k"][e, :, g].double(), x["v"][e, :, g].double()
            s = (q @ k.T) / math.sqrt(d)
            if x["slopes"] is not None:
                s -= float(x["slopes"][h]) * (at[sk - sq:, None] - at[None, :]).abs()
            s[hidden] = -math.inf
            w = torch.softmax(s, 1)
            w[empty] = 0.0
            o = w @ v
            got["out"][e, :, h] = o
            if case["train"]:
                do = x["do"][e, :, h].double()
                dw = do @ v.T
                ds = w * (dw - (w * dw).sum(1, keepdim=True)) / math.sqrt(d)
                got["dq"][e, :, h] = ds @ k
                got["dk"][e, :, g] += ds.T @ q
                got["dv"][e, :, g] += w.T @ do
    return got


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of all batch entries, for one head."""
    sq, sk = case["sq"], case["sk"]
    first = sk - sq
    rows = _documents(case)
    if rows is None:
        one = sum(first + i + 1 for i in range(sq)) if case["causal"] else sq * sk
        return case["b"] * one
    pairs = 0
    for row in rows:  # documents are runs: (start, end) of each
        start = 0
        while start < sk:
            end = start
            while end < sk and row[end] == row[start]:
                end += 1
            if row[start] >= 0:
                low = max(start, first)
                if case["causal"]:
                    pairs += sum(p - start + 1 for p in range(low, end))
                else:
                    pairs += max(0, end - low) * (end - start)
            start = end
    return pairs


def work(case):
    if case["op"] == "attention":
        size, d = _SIZE[case["type"]], case["d"]
        q = case["b"] * case["sq"] * case["hq"] * d
        kv = 2 * case["b"] * case["sk"] * case["hkv"] * d
        flops = 4 * d * case["hq"] * _pairs(case)
        moved = 2 * q + kv
        if case["train"]:  # do read, dq, dk and dv written; five products more
            moved += 2 * q + kv
            flops = flops * 7 // 2
        return {"bytes": moved * size, "flops": flops}
    if case["op"] == "rotary":
        rows = case["b"] * case["s"] * (case["hq"] + case["hkv"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * rows * case["d"] * _SIZE[case["type"]]
                                   + 8 * case["b"] * case["s"]),
                "flops": passes * 3 * rows * case["dim"]}
    parts = _sizes(case)
    n = sum(math.prod(s) for s, _ in parts)
    moved = sum(math.prod(s) * _SIZE[k] for s, k in parts)
    if case["op"] == "norm":
        return {"bytes": moved, "flops": 2 * n}
    return {"bytes": 2 * moved, "flops": 3 * n}
