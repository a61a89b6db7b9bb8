"""Self-attention by its formula in 64 bits, and how far 16-bit operands may move each result."""
import math

import torch


def reference(q, k, v, dout, causal=False, lengths=None, scale=None, store=None):
    """Outputs and gradients {"out", "dq", "dk", "dv"} in 64 bits, and elementwise bounds for the errors of a computation that
    rounds the probabilities, their gradients and the stored results to the type `store`, and accumulates in 32 bits.

    With u the half step of `store` and t its smallest half step (underflow), to first order and with sums of absolute values:
        |P~ - P| <= u P + t                           O: (u P + t) |V| + u |O| + t
        D~ = dO . O~ with the stored O~               dD <= |dO| . bound(O)
        dS~ = P (dP - D~) rounded                     e = u |dS| + t / f + P dD
        dQ: scale e |K| + u |dQ| + t                  dK alike with e^T |Q|, dV: (u P + t / 2^10)^T |dO| + u |dV| + t
    where fp16 holds the backward pass's P times 2^10 and dS times a power of two f with 2^14 <= f 2 d max|dO| max|V| < 2^15
    plus `slack` of the sums of absolute values for the accumulation in 32 bits (2^-24 per term, up to some thousand terms in
    no fixed order), exponentials (2^-22) and exponents (a score of up to 64 in units of log2, rounded, is off by 2^-18)."""
    b, s, h, d = q.shape
    hk = k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    qd, kd, vd, do = (t.detach().double().transpose(1, 2) for t in (q, k, v, dout))
    kd, vd = (t.repeat_interleave(h // hk, 1) for t in (kd, vd))
    pos = torch.arange(s, device=q.device)
    n = torch.full((b,), s, device=q.device) if lengths is None else lengths.clamp(0, s)
    rows = (pos[None] < n[:, None])[:, None, :, None]
    qd, kd, vd, do = (torch.where(rows, t, 0.0) for t in (qd, kd, vd, do))
    valid = rows & rows.transpose(2, 3)
    if causal:
        valid = valid & (pos[None, :] <= pos[:, None])
    x = (qd @ kd.mT) * scale
    x = torch.where(valid, x, -math.inf)
    x = torch.exp(x - torch.where(rows, x.amax(-1, keepdim=True), 0.0))
    p = x / torch.where(rows, x.sum(-1, keepdim=True), 1.0)
    out = p @ vd
    dp = do @ vd.mT
    ds = p * (dp - (dp * p).sum(-1, keepdim=True))

    def fold(t):  # sum of a group's heads
        return t.reshape(b, hk, h // hk, s, d).sum(2)

    want = {"out": out, "dq": ds @ kd * scale, "dk": fold(ds.mT @ qd) * scale, "dv": fold(p.mT @ do)}
    want = {name: t.transpose(1, 2) for name, t in want.items()}
    store = q.dtype if store is None else store
    u = torch.finfo(store).eps / 2
    t = 2.0 ** -25 if store == torch.float16 else 0.0
    slack = 2.0 ** -14
    pe = (u + slack) * p + t * valid
    oe = pe @ vd.abs() + u * out.abs() + t
    mag = p * (do.abs() @ vd.abs().mT + (do.abs() * out.abs()).sum(-1, keepdim=True))
    most = 2 * d * do.abs().reshape(b, hk, -1).amax(-1) * vd.abs().reshape(b, hk, -1).amax(-1)
    f = (2.0 ** 14 / most.clamp_min(1e-30)).repeat_interleave(h // hk, 1)[:, :, None, None]
    e = u * ds.abs() + slack * mag + t / f * valid + p * (do.abs() * oe).sum(-1, keepdim=True)
    pb = (u + slack) * p + t / 1024 * valid
    bound = {"out": oe, "dq": e @ kd.abs() * scale, "dk": fold(e.mT @ qd.abs()) * scale, "dv": fold(pb.mT @ do.abs())}
    bound = {name: x.transpose(1, 2) for name, x in bound.items()}
    for name in ("dq", "dk", "dv"):
        bound[name] = bound[name] + u * want[name].abs() + t
    return want, bound


def check(got, want, bound):
    for name, x in got.items():
        off = (x.double() - want[name]).abs()
        worst = (off / bound[name].clamp_min(1e-300)).nan_to_num(nan=math.inf if not x.isfinite().all() else 0.0)
        worst = torch.where(off == 0, 0.0, worst)
        assert bool((off <= bound[name]).all()), f"{name}: {float(worst.max()):.3g} times its bound"
