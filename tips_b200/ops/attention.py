"""Self-attention without layout glue.

``attention(q, k, v)`` is this package's own attention (csrc/kernels/attention.cu): causal or padded batches, shared key and
value heads, forward and a backward pass that recomputes the probabilities.

``packed_attention(qkv, heads)`` takes the output of the fused QKV linear layer, ``[batch, seq, 3 * hidden]``, and
returns ``[batch, seq, hidden]``.  With ``kv_heads``, ``lengths`` or ``scale`` it runs ``attention`` on views of the packed
tensor.  Without them the attention itself is the library's fused scaled-dot-product attention (the
reference has no attention at all; its models are TensorFlow's), but everything around it is done here so that
no tensor is re-laid by generic strided copies: q, k and v are strided views of the packed tensor, the output and
the incoming gradient change layout with one vectorised pass of ``tipsk_copy4d`` each.  Either way the three gradients
are written straight into one packed ``[batch, seq, 3, heads, d]`` buffer (instead of three zero-filled tensors that
autograd then sums).
"""
from __future__ import annotations

import ctypes
import math

import torch
import torch.nn.functional as F

from . import base


def copy4d(src: torch.Tensor, dst: torch.Tensor) -> None:
    """dst[...] = src[...] for 4-D tensors of equal shape whose last axis is contiguous on both sides."""
    assert src.shape == dst.shape and src.dim() == 4 and src.dtype == dst.dtype
    assert src.stride(3) == 1 and dst.stride(3) == 1
    es = src.element_size()
    n0, n1, n2, d = src.shape
    ss = (ctypes.c_int64 * 3)(*(src.stride(i) * es for i in range(3)))
    ds = (ctypes.c_int64 * 3)(*(dst.stride(i) * es for i in range(3)))
    base.check(base.K().tipsk_copy4d(src.data_ptr(), dst.data_ptr(), n0, n1, n2, d * es, ss, ds, base.stream()),
               "copy4d")


def _fast_ok(t: torch.Tensor, d: int) -> bool:
    return t.is_cuda and t.dtype in (torch.bfloat16, torch.float16) and (d * t.element_size()) % 16 == 0


class _PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, heads, causal):
        b, s, three_h = qkv.shape
        h = three_h // 3
        d = h // heads
        packed = qkv.detach().view(b, s, 3, heads, d)
        with torch.enable_grad():
            q, k, v = (packed[:, :, i].transpose(1, 2).requires_grad_() for i in range(3))  # [b, heads, s, d] views
            out = F.scaled_dot_product_attention(q, k, v, is_causal=causal)
        ctx.graph = (q, k, v, out)
        ctx.geom = (b, s, heads, d)
        o = out.detach()
        if o.transpose(1, 2).is_contiguous():  # the library kept the [b, s, heads, d] memory order of the inputs
            return o.transpose(1, 2).reshape(b, s, h)
        y = torch.empty(b, s, heads, d, dtype=o.dtype, device=o.device)
        copy4d(o.transpose(1, 2), y)
        return y.view(b, s, h)

    @staticmethod
    def backward(ctx, dy):
        q, k, v, out = ctx.graph
        b, s, heads, d = ctx.geom
        ctx.graph = None
        dyv = dy.reshape(b, s, heads, d)
        if out.transpose(1, 2).is_contiguous():
            dout = dyv.transpose(1, 2)  # same memory order as `out`
        else:
            dout = torch.empty(b, heads, s, d, dtype=dy.dtype, device=dy.device)
            copy4d(dyv.transpose(1, 2), dout)
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
        dqkv = torch.empty(b, s, 3, heads, d, dtype=dy.dtype, device=dy.device)
        for i, g in enumerate((dq, dk, dv)):
            copy4d(g.transpose(1, 2), dqkv[:, :, i])  # [b, s, heads, d] view of the gradient -> its packed slot
        return dqkv.view(b, s, 3 * heads * d), None, None


def _check_lengths(lengths, b: int, device) -> None:
    if lengths is None:
        return
    if not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError("lengths must be an int32 or int64 tensor")
    if tuple(lengths.shape) != (b,):
        raise ValueError(f"lengths must have one entry per sequence: shape ({b},), got {tuple(lengths.shape)}")
    if lengths.device != device:
        raise ValueError(f"lengths are on {lengths.device}, the inputs on {device}")


def _check_attention(t, s, h, hk, d, lengths, scale) -> float:
    """Checks sizes, type and the other arguments of an attention over a tensor like `t` and returns the scale to use."""
    if h <= 0 or hk <= 0 or h % hk != 0:
        raise ValueError(f"{h} heads cannot share {hk} key and value heads evenly")
    if d <= 0:
        raise ValueError("the head size must be positive")
    if not t.dtype.is_floating_point:
        raise TypeError(f"attention takes floating-point tensors, got {t.dtype}")
    _check_lengths(lengths, t.shape[0], t.device)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if t.is_cuda:
        if t.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"attention on a GPU takes bfloat16 or float16, got {t.dtype}")
        if d % 8 != 0 or d > 128:
            raise ValueError(f"attention on a GPU takes head sizes that are multiples of 8 up to 128, got {d}")
        b, group = t.shape[0], h // hk
        if b * s > 0 and (b > 65535 or h > 1 << 17 or s * group > 1 << 25 or b * (h + hk) * -(-s // 128) >= 1 << 31):
            raise ValueError("attention on a GPU takes up to 65535 sequences, 2**17 heads, 2**25 positions times query heads per key head "
                             f"and 2**31 tiles of 128 positions of a head, got {b} sequences of {s} with {h} heads and {hk} key heads")
        if not 2.0 ** -149 <= scale <= 2.3e38:
            raise ValueError(f"scale must be within the range of 32 bits, got {scale}")
    return scale


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where the kernels cannot read it in place: they need a contiguous last axis, positive strides of whole
    16 bytes and a 16-byte-aligned start."""
    sb, ss, sh, sd = t.stride()
    if sd == 1 and t.data_ptr() % 16 == 0 and sb > 0 and ss > 0 and sh > 0 and (sb | ss | sh) % 8 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _view(t: torch.Tensor):
    """(address, strides) of a [batch, seq, heads, d] tensor as the launchers take them."""
    return t.data_ptr(), t.stride()[:3]


def _heads_view(t: torch.Tensor, shape):
    """The same of the query heads in a tensor of that shape, or in a contiguous [batch, seq, heads * d] one."""
    if t.dim() == 4:
        return _view(t)
    _, s, h, _, d = shape
    return t.data_ptr(), (s * h * d, h * d, d)


def _packed_views(t: torch.Tensor, h: int, hk: int, d: int):
    """The same of the q, k and v heads of a contiguous [batch, seq, (h + 2 hk) * d] tensor, without making views."""
    at, row, step = t.data_ptr(), (h + 2 * hk) * d, d * t.element_size()
    st = (t.shape[1] * row, row, d)
    return (at, st), (at + h * step, st), (at + (h + hk) * step, st)


def _strides(*views):
    return base.i64_array([x for _, st in views for x in st])


def _lse_bytes(shape) -> int:
    b, s, h, _, _ = shape
    return b * h * (-(-s // 128) * 128) * 4


def _rest_bytes(shape, lengths, causal) -> int:
    """Bytes for what the rounding of the output drops in rows of up to 128 keys, if there can be any."""
    b, s, h, _, d = shape
    return b * min(s, 128) * h * d if causal or lengths is not None or s <= 128 else 0


def _attention_fwd(like, shape, q, k, v, lengths, scale, causal, grad=True, flat=False):
    """(out, stats) for the views q, k, v of CUDA tensors like `like`; shape = (b, s, h, hk, d), `flat`: out is [b, s, h * d].  `stats`: bytes of the rows'
    log-sums and, for a backward pass to come, what rounding dropped of `out` in rows of few keys."""
    b, s, h, hk, d = shape
    out = torch.empty((b, s, h * d) if flat else (b, s, h, d), dtype=like.dtype, device=like.device)
    at, rest = _lse_bytes(shape), _rest_bytes(shape, lengths, causal) if grad else 0
    stats = torch.empty(at + rest, dtype=torch.uint8, device=like.device)
    if out.numel():
        with base.device_of(like):
            base.check(base.K().tipsk_attention_fwd(
                q[0], k[0], v[0], out.data_ptr(), stats.data_ptr(), stats.data_ptr() + at if rest else None, base.ptr(lengths),
                int(lengths is not None and lengths.dtype == torch.int64), b, s, h, hk, d, base.code(like),
                _strides(q, k, v, _heads_view(out, shape)), scale, int(causal), base.stream()), "attention_fwd")
    return out, stats


def _attention_bwd(dout, shape, q, k, v, out, stats, lengths, scale, causal, dq, dk, dv):
    """Writes the gradients into the views dq, dk, dv."""
    b, s, h, hk, d = shape
    if not out.numel():
        return
    dout = _rows16(dout) if dout.dim() == 4 else _packed16(dout)
    at = _lse_bytes(shape)
    delta = torch.empty(at // 2 + 2 * b * hk, dtype=torch.float32, device=out.device)
    with base.device_of(out):
        base.check(base.K().tipsk_attention_bwd(
            dout.data_ptr(), q[0], k[0], v[0], out.data_ptr(), stats.data_ptr(), stats.data_ptr() + at if _rest_bytes(shape, lengths, causal) else None,
            delta.data_ptr(), dq[0], dk[0], dv[0],
            base.ptr(lengths), int(lengths is not None and lengths.dtype == torch.int64), b, s, h, hk, d, base.code(out),
            _strides(q, k, v, _heads_view(out, shape), _heads_view(dout, shape), dq, dk, dv), scale, int(causal), base.stream()), "attention_bwd")
    base.count_launches(1)


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, scale, causal, grad):
        shape = (*q.shape[:3], k.shape[2], q.shape[3])
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        out, stats = _attention_fwd(q, shape, _view(q), _view(k), _view(v), lengths, scale, causal, grad)
        ctx.save_for_backward(q, k, v, out, stats, lengths)
        ctx.meta = (shape, scale, causal)
        return out

    @staticmethod
    @base.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, stats, lengths = ctx.saved_tensors
        shape, scale, causal = ctx.meta
        # a saved-tensor hook may have changed the layout
        q, k, v, out, stats = _rows16(q), _rows16(k), _rows16(v), _rows16(out), _packed16(stats)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        _attention_bwd(dout, shape, _view(q), _view(k), _view(v), out, stats, lengths, scale, causal, _view(dq), _view(dk), _view(dv))
        return dq, dk, dv, None, None, None, None


def _packed16(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _PackedOwnAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, h, hk, lengths, scale, causal, grad):
        qkv = _packed16(qkv)
        b, s, width = qkv.shape
        shape = (b, s, h, hk, width // (h + 2 * hk))
        out, stats = _attention_fwd(qkv, shape, *_packed_views(qkv, h, hk, shape[4]), lengths, scale, causal, grad, flat=True)
        ctx.save_for_backward(qkv, out, stats, lengths)
        ctx.meta = (shape, scale, causal)
        return out

    @staticmethod
    @base.once_differentiable
    def backward(ctx, dy):
        qkv, out, stats, lengths = ctx.saved_tensors
        shape, scale, causal = ctx.meta
        _, _, h, hk, d = shape
        qkv, out, stats = _packed16(qkv), _packed16(out), _packed16(stats)
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _attention_bwd(dy, shape, *_packed_views(qkv, h, hk, d), out, stats, lengths, scale, causal,
                       *_packed_views(dqkv, h, hk, d))
        return dqkv, None, None, None, None, None, None


def attention_status() -> int:
    """0 when no attention launch on the current device since the last call reported a bounded-wait timeout
    (waits for all of its streams)."""
    return int(base.K().tipsk_attention_status())


def _plain_attention(q, k, v, lengths, scale, causal):
    """The formula, for CPU tensors."""
    b, s, h, d = q.shape
    group = h // k.shape[2]
    qf, kf, vf = ((t if t.dtype == torch.float64 else t.float()).transpose(1, 2) for t in (q, k, v))
    kf, vf = kf.repeat_interleave(group, 1), vf.repeat_interleave(group, 1)
    pos = torch.arange(s, device=q.device)
    rows = torch.ones(b, s, dtype=torch.bool, device=q.device)
    if lengths is not None:
        rows = pos[None] < lengths[:, None]
        # what stands beyond a length must not count, whatever it is
        qf, kf, vf = (torch.where(rows[:, None, :, None], t, 0.0) for t in (qf, kf, vf))
    valid = rows[:, None, None, :]
    if causal:
        valid = valid & (pos[None, :] <= pos[:, None])
    logits = (qf @ kf.transpose(-1, -2)) * scale
    # a row without any valid key: zeros, by way of a softmax over all keys whose result is dropped
    logits = logits.masked_fill(~valid & rows[:, None, :, None], -math.inf)
    out = torch.where(rows[:, None, :, None], torch.softmax(logits, -1) @ vf, 0.0)
    return out.transpose(1, 2).to(q.dtype)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False, lengths: torch.Tensor | None = None,
              scale: float | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v for ``q [batch, seq, heads, d]`` and ``k, v [batch, seq, kv_heads, d]``; returns
    ``[batch, seq, heads, d]``.

    `kv_heads` divides `heads`: query head i reads key and value head ``i // (heads // kv_heads)``.  `causal`: a position sees
    itself and what is before it.  `lengths` (int32 or int64 ``[batch]``, on the inputs' device): the positions of a sequence
    from its length on are padding.  They are not read as keys or values, their rows of the output are zero, and so are their
    gradients, whatever stands in them; a length outside 0..seq counts as the nearer of the two.  `scale` (positive) defaults
    to ``1 / sqrt(d)``.

    On a GPU: bfloat16 or float16, d a multiple of 8 up to 128, any strides (inputs whose last axis is not contiguous, or
    whose rows do not start on 16 bytes, are copied), up to 65535 sequences, 2**17 heads, and 2**25 for seq times the query
    heads of a key head.  The softmax is held in fp32; the probabilities, and their gradient in the backward pass, are rounded
    to the inputs' type as operands of the products (for float16 at a scale that keeps them within its range; the gradient as a
    sum of two values where seq is at most 128).  Gradients do not depend on the order of the blocks.  An infinity or NaN in a
    valid position may reach every row of a causal batch, also those that do not see it, as 0 * inf does in the formula.
    `lengths` may not change between forward and backward."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be [batch, seq, heads, head_size], got {tuple(t.shape)}")
        if t.dtype != q.dtype or t.device != q.device:
            raise TypeError(f"q, k and v must share dtype and device: {name} is {t.dtype} on {t.device}, q {q.dtype} on {q.device}")
    b, s, h, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[1] != s or k.shape[3] != d:
        raise ValueError(f"k and v must be [{b}, {s}, kv_heads, {d}] like q, got {tuple(k.shape)} and {tuple(v.shape)}")
    scale = _check_attention(q, s, h, k.shape[2], d, lengths, scale)
    if not q.is_cuda:
        return _plain_attention(q, k, v, lengths, scale, causal)
    if lengths is not None:
        lengths = lengths.contiguous()
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _AttentionFn.apply(q, k, v, lengths, scale, bool(causal), grad)


def packed_attention(qkv: torch.Tensor, heads: int, causal: bool = False, kv_heads: int | None = None,
                     lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Multi-head self-attention on ``qkv = [batch, seq, 3 * hidden]`` (q, k, v concatenated on the last axis).

    With any of `kv_heads`, `lengths`, `scale` it is `attention` (see there) on the heads of the packed tensor, whose last axis
    holds ``heads`` heads of q and then `kv_heads` (default: `heads`) heads of k and of v."""
    if kv_heads is not None or lengths is not None or scale is not None:
        hk = heads if kv_heads is None else kv_heads
        if qkv.dim() != 3 or heads <= 0 or hk <= 0 or qkv.shape[2] == 0 or qkv.shape[2] % (heads + 2 * hk) != 0:
            raise ValueError(f"qkv must be [batch, seq, ({heads} + 2 * {hk}) * head_size], got {tuple(qkv.shape)}")
        b, s, width = qkv.shape
        scale = _check_attention(qkv, s, heads, hk, width // (heads + 2 * hk), lengths, scale)
        if not qkv.is_cuda:
            x = qkv.view(b, s, heads + 2 * hk, -1) if b and s else qkv.new_empty(b, s, heads + 2 * hk, width // (heads + 2 * hk))
            return _plain_attention(*x.split([heads, hk, hk], 2), lengths, scale, causal).reshape(b, s, -1)
        if lengths is not None:
            lengths = lengths.contiguous()
        return _PackedOwnAttentionFn.apply(qkv, heads, hk, lengths, scale, bool(causal), torch.is_grad_enabled() and qkv.requires_grad)
    b, s, three_h = qkv.shape
    d = three_h // 3 // heads
    if _fast_ok(qkv, d) and qkv.is_contiguous():
        return _PackedAttentionFn.apply(qkv, heads, causal)
    q, k, v = qkv.view(b, s, 3, heads, d).permute(2, 0, 3, 1, 4)
    att = F.scaled_dot_product_attention(q, k, v, is_causal=causal)
    return att.transpose(1, 2).reshape(b, s, three_h // 3)
