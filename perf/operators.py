"""Operators of a transformer's training step: what is timed, in plain form and through this framework's entry points.

    attention     self-attention on a padded or causal batch, forward and backward (the probabilities are recomputed)
    attention_fwd the same without gradients
    pack          a tensor stored in 8 bits with a power-of-two step per 32 values, and read back
    linear        a dense layer that keeps its activations for the backward pass in 8 bits, forward and backward

Sizes are those of the BERT-shaped encoder of this repository (hidden 1024, 16 heads, sequences of 512, feed-forward 4096; its
small test model), of its click model's dense layers, and generic ones around them.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the small test encoder: two sequences of 64 tokens, latency of a few launches
        {"name": "attn_2x64_h4_d32", "kind": "attention", "dtype": "bf16", "batch": 2, "seq": 64, "heads": 4, "kv_heads": 4, "dim": 32,
         "causal": False, "lengths": "full", "packed": True},
        # the pre-training batch of the encoder, padded to 512 tokens
        {"name": "attn_32x512_h16_d64", "kind": "attention", "dtype": "bf16", "batch": 32, "seq": 512, "heads": 16, "kv_heads": 16, "dim": 64,
         "causal": False, "lengths": "ragged", "packed": True},
        # a causal model with shared key and value heads
        {"name": "attn_2x2048_h16_kv4_d128", "kind": "attention", "dtype": "bf16", "batch": 2, "seq": 2048, "heads": 16, "kv_heads": 4, "dim": 128,
         "causal": True, "lengths": "none", "packed": False},
        # one long causal sequence
        {"name": "attn_1x8192_h16_kv4_d128", "kind": "attention", "dtype": "bf16", "batch": 1, "seq": 8192, "heads": 16, "kv_heads": 4, "dim": 128,
         "causal": True, "lengths": "none", "packed": False},
        # odd lengths, some of them zero, a head size between the tiles', fp16
        {"name": "attn_5x777_h12_d80_fp16", "kind": "attention", "dtype": "fp16", "batch": 5, "seq": 777, "heads": 12, "kv_heads": 12, "dim": 80,
         "causal": False, "lengths": "holes", "packed": False},
        # evaluation of the encoder on a padded batch
        {"name": "attn_fwd_32x512_h16_d64", "kind": "attention_fwd", "dtype": "bf16", "batch": 32, "seq": 512, "heads": 16, "kv_heads": 16, "dim": 64,
         "causal": False, "lengths": "ragged", "packed": True},
        # a small activation of odd size in fp32
        {"name": "pack_37x101_fp32", "kind": "pack", "dtype": "fp32", "rows": 37, "cols": 101},
        # the feed-forward activation of the pre-training batch
        {"name": "pack_16384x4096", "kind": "pack", "dtype": "bf16", "rows": 16384, "cols": 4096},
        # feed-forward layer of the pre-training batch: input and pre-activation kept in 8 bits
        {"name": "linear8_16384x1024x4096_gelu", "kind": "linear", "dtype": "bf16", "rows": 16384, "k": 1024, "n": 4096, "act": "gelu"},
        # the layer behind it: input kept in 8 bits, no activation
        {"name": "linear8_16384x4096x1024", "kind": "linear", "dtype": "bf16", "rows": 16384, "k": 4096, "n": 1024, "act": "none"},
        # the small test encoder's layer on few rows
        {"name": "linear8_128x128x512_gelu", "kind": "linear", "dtype": "bf16", "rows": 128, "k": 128, "n": 512, "act": "gelu"},
        # a ragged row count and widths of no tile's size
        {"name": "linear8_2311x520x1096_gelu", "kind": "linear", "dtype": "bf16", "rows": 2311, "k": 520, "n": 1096, "act": "gelu"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention_fwd", "pack", "linear", "linear"])
    if kind in ("attention", "attention_fwd"):
        kv_heads, group = rng.choice([(1, 8), (2, 4), (4, 1), (4, 4), (8, 2), (12, 1), (16, 1), (3, 5)])
        heads = kv_heads * group
        batch = _log(rng, 1, 32)
        most = math.sqrt(16 * 8192 * 8192 / (batch * heads))
        seq = _log(rng, 16, min(8192.0, most))
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
                "dim": rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128]), "causal": rng.random() < 0.5,
                "lengths": rng.choice(["none", "ragged", "holes"]), "packed": rng.random() < 0.5}
    if kind == "pack":
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": _log(rng, 1, 16384), "cols": _log(rng, 8, 4096)}
    return {"kind": kind, "dtype": "bf16", "rows": _log(rng, 64, 16384), "k": 8 * _log(rng, 8, 256), "n": 8 * _log(rng, 8, 256),
            "act": rng.choice(["none", "gelu", "gelu"])}


# ---- inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] in ("attention", "attention_fwd"):
        b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
        if case["packed"]:  # one projection's output: q heads, k heads, v heads on the last axis
            inputs = (_randn(g, (b, s, (h + 2 * hk) * d), dt),)
        else:
            inputs = tuple(_randn(g, (b, s, n, d), dt) for n in (h, hk, hk))
        dout = _randn(g, (b, s, h * d) if case["packed"] else (b, s, h, d), dt)
        lengths = None
        if case["lengths"] != "none":
            lengths = torch.randint(1, s + 1, (b,), generator=g, device=DEV)
            lengths[0] = s
            if case["lengths"] == "full":
                lengths.fill_(s)
            if case["lengths"] == "holes":
                lengths[1::3] = 0
        train = case["kind"] == "attention"
        return {"case": case, "inputs": [t.requires_grad_(train) for t in inputs], "dout": dout, "lengths": lengths}
    if case["kind"] == "pack":
        x = _randn(g, (case["rows"], case["cols"]), torch.float32)
        # activations: most values small, a few channels far larger
        x = x * torch.exp(torch.randn(case["cols"], generator=g, device=DEV))
        return {"case": case, "x": x.to(dt)}
    m, k, n = case["rows"], case["k"], case["n"]
    leaf = lambda t: t.requires_grad_(True)  # noqa: E731
    return {"case": case, "x": leaf(_randn(g, (m, k), dt)), "w": leaf(_randn(g, (n, k), dt, 1.0 / math.sqrt(k))), "b": leaf(_randn(g, (n,), dt, 0.1)),
            "dy": _randn(g, (m, n), dt)}


def _heads(case, inputs):
    """q, k, v as [batch, seq, heads, dim] views of the case's inputs."""
    if not case["packed"]:
        return inputs
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    x = inputs[0].view(case["batch"], case["seq"], h + 2 * hk, d)
    return x[:, :, :h], x[:, :, h:h + hk], x[:, :, h + hk:]


# ---- plain forms: elementary operations in 32 bits, rounded once


def _plain_attention(case, state):
    dt = DTYPES[case["dtype"]]
    b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    group = h // hk
    q, k, v = (t.detach().float().transpose(1, 2) for t in _heads(case, state["inputs"]))  # [b, heads, s, d]
    q = q.reshape(b, hk, group, s, d)
    k, v = k.unsqueeze(2), v.unsqueeze(2)
    at = torch.arange(s, device=DEV)
    valid = torch.ones(b, 1, 1, s, s, dtype=torch.bool, device=DEV)
    rows = torch.ones(b, 1, 1, s, 1, dtype=torch.bool, device=DEV)
    if state["lengths"] is not None:
        inside = at[None, :] < state["lengths"][:, None]
        rows = inside[:, None, None, :, None]
        valid = valid & rows & inside[:, None, None, None, :]
    if case["causal"]:
        valid = valid & (at[None, :] <= at[:, None])
    scale = 1.0 / math.sqrt(d)
    p = (q @ k.transpose(-1, -2)) * scale
    p = torch.where(valid, p, torch.full((), -math.inf, device=DEV))
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(rows, top, torch.zeros((), device=DEV)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(rows, total, torch.ones((), device=DEV))
    out = p @ v

    def back(t, n):  # [b, ..., s, d] -> the layout of the caller
        return t.reshape(b, n, s, d).transpose(1, 2)

    y = back(out, h).to(dt)
    y = y.reshape(b, s, h * d) if case["packed"] else y.contiguous()
    if case["kind"] == "attention_fwd":
        return y
    do = state["dout"].float().view(b, s, h, d).transpose(1, 2).reshape(b, hk, group, s, d)
    do = torch.where(rows, do, torch.zeros((), device=DEV))
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = do @ v.transpose(-1, -2)
    ds = p * (ds - (ds * p).sum(-1, keepdim=True))
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2) * scale
    grads = [back(dq, h).to(dt), back(dk, hk).to(dt), back(dv, hk).to(dt)]
    if case["packed"]:
        return y, torch.cat(grads, 2).reshape(b, s, (h + 2 * hk) * d)
    return y, [t.contiguous() for t in grads]


def _plain_pack(x):
    """x in 32 bits -> the values that its 8-bit form stands for, in 32 bits."""
    n = x.numel()
    flat = torch.zeros((n + 31) // 32 * 32, dtype=torch.float32, device=x.device)
    flat[:n] = x.reshape(-1)
    flat = flat.view(-1, 32)
    part, power = torch.frexp(flat.abs().amax(1, keepdim=True))
    e = power - 7 + (part * 128 >= 127.5).to(power.dtype)
    e = torch.where(part == 0, torch.full_like(e, -126), e.clamp(-126, 121))
    step = ((e + 127) << 23).view(torch.float32)  # 2^e by its bits: powers computed otherwise may be an ulp off, which breaks ties
    return (torch.round(flat / step).clamp(-127, 127) * step).view(-1)[:n].view(x.shape)


def _plain_linear(case, state):
    dt = DTYPES[case["dtype"]]
    x, w, b = (state[n].detach().float() for n in ("x", "w", "b"))
    pre = x @ w.t() + b
    kept_x = _plain_pack(x)
    dz = state["dy"].float()
    if case["act"] == "gelu":
        y = pre * 0.5 * (1 + torch.erf(pre / math.sqrt(2)))
        z = _plain_pack(pre.to(dt).float())  # the layer keeps what its input type holds
        dz = dz * (0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    else:
        y = pre
    return y.to(dt), (dz @ w).to(dt), (dz.t() @ kept_x).to(dt), dz.sum(0).to(dt)


# ---- the pass


def _own_attention(case, state):
    from tips_b200.ops.attention import attention, packed_attention
    if case["packed"]:
        y = packed_attention(state["inputs"][0], case["heads"], case["causal"], kv_heads=case["kv_heads"], lengths=state["lengths"])
    else:
        y = attention(*state["inputs"], causal=case["causal"], lengths=state["lengths"])
    if case["kind"] == "attention_fwd":
        return y
    grads = torch.autograd.grad(y, state["inputs"], state["dout"])
    return (y.detach(), grads[0]) if case["packed"] else (y.detach(), list(grads))


def _own_linear(case, state):
    from tips_b200.ops.linear import linear
    y = linear(state["x"], state["w"], state["b"], case["act"], save8=True)
    return (y.detach(), *torch.autograd.grad(y, (state["x"], state["w"], state["b"]), state["dy"]))


def _own_pack(case, state):
    from tips_b200.ops.saved8 import pack8
    return pack8(state["x"]).unpack()


def run(state):
    case = state["case"]
    if case["kind"] in ("attention", "attention_fwd"):
        return _own_attention(case, state) if own else _plain_attention(case, state)
    if case["kind"] == "pack":
        return _own_pack(case, state) if own else _plain_pack(state["x"].float()).to(state["x"].dtype)
    return _own_linear(case, state) if own else _plain_linear(case, state)


# ---- what a pass cannot do without


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "pack":
        n = case["rows"] * case["cols"]
        return {"bytes": n * es * 2 + 2 * (n + (n + 31) // 32), "flops": 0}  # read, stored in 8 bits, read again, written
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        values = 2 * m * k + 2 * m * n + 2 * n * k + 2 * n  # x, dx, y, dy, w, dw, b, db
        kept = m * k + (m * n if case["act"] == "gelu" else 0)
        return {"bytes": es * values + 2 * (kept + kept // 32), "flops": 3 * 2 * m * n * k}
    b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    # ragged lengths are uniform on 1..s with the first one full; every third is empty with holes
    if case["lengths"] in ("none", "full"):
        tokens, pairs = b * s, b * s * s
    else:
        empty = len(range(1, b, 3)) if case["lengths"] == "holes" else 0
        rest = b - 1 - empty
        tokens, pairs = s + rest * (s + 1) / 2, s * s + rest * (s + 1) * (2 * s + 1) / 6
    if case["causal"]:
        pairs = (pairs + tokens) / 2
    train = case["kind"] == "attention"
    read = (h + 2 * hk + (2 * h if train else 0)) * d * tokens  # q, k, v; the output and its gradient in the backward pass
    written = (h + (h + 2 * hk if train else 0)) * d * b * s
    return {"bytes": int(es * (read + written)), "flops": int((7 if train else 2) * 2 * h * d * pairs)}


# ---- definitions in 64 bits


def _exact_pack(x):
    n = x.numel()
    flat = torch.nn.functional.pad(x.double().reshape(-1), (0, -n % 32)).view(-1, 32)
    amax = flat.abs().max(1, keepdim=True).values
    # the least e with amax / 2^e < 127.5
    e = torch.floor(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / 127.5)) + 1
    e = torch.where(amax > 0, e.clamp(-126, 121), torch.full_like(e, -126))
    step = ((e.long() + 1023) << 52).view(torch.float64)  # 2^e exactly
    return ((flat / step).round().clamp(-127, 127) * step).view(-1)[:n].view(x.shape)


def _exact_attention(case, state):
    h, hk, d, s = case["heads"], case["kv_heads"], case["dim"], case["seq"]
    dev = state["dout"].device
    lengths = state["lengths"] if state["lengths"] is not None else torch.full((case["batch"],), s, device=dev)
    train = case["kind"] == "attention"
    out, grads = [], []
    for i, inputs in enumerate(zip(*(t.detach() for t in state["inputs"]))):  # sequence by sequence
        n = int(lengths[i])
        leaves = [t.double().requires_grad_(train) for t in inputs]
        x = leaves if not case["packed"] else leaves[0].view(s, h + 2 * hk, d).split([h, hk, hk], 1)
        q, k, v = x[0][:n], x[1][:n].repeat_interleave(h // hk, 1), x[2][:n].repeat_interleave(h // hk, 1)
        logits = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(d)
        if case["causal"]:
            logits = logits + torch.full((n, n), -math.inf, dtype=torch.float64, device=dev).triu(1)
        o = torch.einsum("hij,jhd->ihd", logits.softmax(-1), v)
        out.append(torch.nn.functional.pad(o.detach().reshape(n, h * d), (0, 0, 0, s - n)))
        if train:
            do = state["dout"][i, :n].double().view(n, h, d)
            grads.append(torch.autograd.grad((o * do).sum(), leaves))
    y = torch.stack(out)
    y = y if case["packed"] else y.view(case["batch"], s, h, d)
    if not train:
        return y
    grads = [torch.stack(g) for g in zip(*grads)]
    return (y, grads[0]) if case["packed"] else (y, grads)


def _exact_linear(case, state):
    x, w, b = (state[n].detach().double() for n in ("x", "w", "b"))
    pre = torch.addmm(b, x, w.t())
    g = state["dy"].double()
    y = pre
    if case["act"] == "gelu":
        phi = torch.distributions.Normal(0.0, 1.0)
        y = pre * phi.cdf(pre)
        z = _exact_pack(pre.to(DTYPES[case["dtype"]]))
        g = g * (phi.cdf(z) + z * phi.log_prob(z).exp())
    return y, g @ w, g.t() @ _exact_pack(x), g.sum(0)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "pack":
        return _exact_pack(state["x"])
    return _exact_linear(case, state) if case["kind"] == "linear" else _exact_attention(case, state)
