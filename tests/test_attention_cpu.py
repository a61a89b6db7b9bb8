"""Attention on CPU tensors, and the refusals that need no GPU."""
import ctypes
import math

import pytest
import torch

from attention_util import reference
from tips_b200.ops.attention import attention, packed_attention


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [None, [0, 1, 9], [9, 4, 20]])
def test_formula(causal, lengths):
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(3, 9, n, 6, generator=g) for n in (4, 2, 2, 4))
    n = None if lengths is None else torch.tensor(lengths)
    want, _ = reference(q, k, v, do, causal, n)
    if n is not None:
        for i, m in enumerate(lengths):
            for t in (q, k, v):
                t[i, m:] = math.nan
    leaves = [t.requires_grad_() for t in (q, k, v)]
    y = attention(*leaves, causal=causal, lengths=n)
    got = [y.detach(), *torch.autograd.grad(y, leaves, do)]
    for x, name in zip(got, ("out", "dq", "dk", "dv")):
        assert torch.allclose(x.double(), want[name], rtol=1e-4, atol=1e-5), name
    packed = torch.cat([t.detach().flatten(2) for t in (q, k, v)], 2)
    z = packed_attention(packed, 4, causal, kv_heads=2, lengths=n)
    assert torch.equal(z, y.detach().flatten(2))


def test_refusals():
    x = torch.zeros(2, 5, 4, 8)
    for bad in (dict(k=x[:, :4]), dict(k=x[:1]), dict(v=x[..., :4]), dict(k=x[:, :, :3], v=x[:, :, :3]), dict(k=x[0], v=x[0])):
        with pytest.raises(ValueError):
            attention(**{"q": x, "k": x, "v": x, **bad})
    with pytest.raises(TypeError):
        attention(x, x.double(), x)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            attention(x, x, x, scale=scale)
    for n, kind in ((torch.tensor([1.0, 2.0]), TypeError), ([1, 2], TypeError), (torch.tensor([1]), ValueError),
                    (torch.tensor([[1, 2]]), ValueError)):
        with pytest.raises(kind):
            attention(x, x, x, lengths=n)
    for heads, kv in ((0, None), (4, 0), (4, 3), (5, None), (-2, None)):
        with pytest.raises(ValueError):
            packed_attention(torch.zeros(2, 5, 96), heads, kv_heads=kv, scale=1.0)


def test_the_library_refuses_before_it_reads():
    """Sizes, strides and alignment that the kernels do not take come back as errors of the C entries, without a device."""
    from tips_b200 import _lib
    if not _lib.kernels_available():
        pytest.skip("kernel library not built")
    lib = _lib.kernels()
    ok = dict(b=1, s=16, h=2, hk=2, d=64, dtype=6, scale=0.125)
    strides = (ctypes.c_int64 * 12)(*[2048, 128, 64] * 4)

    def call(at=4096, strides=strides, **kw):
        a = {**ok, **kw}
        return lib.tipsk_attention_fwd(at, at, at, at, at, None, None, 0, a["b"], a["s"], a["h"], a["hk"], a["d"], a["dtype"], strides,
                                       a["scale"], 0, None)

    for kw in (dict(d=0), dict(d=12), dict(d=136), dict(hk=3), dict(h=0), dict(hk=0), dict(b=0), dict(s=0), dict(dtype=0),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=3e38), dict(s=1 << 30, b=1 << 10), dict(h=1 << 18, hk=1 << 18), dict(s=(1 << 24) + 1, h=4, hk=2),
               dict(at=4100)):
        assert call(**kw) == -2, kw
    for i, x in ((1, 132), (3, 0), (8, -64), (11, 4)):
        bad = (ctypes.c_int64 * 12)(*strides)
        bad[i] = x
        assert call(strides=bad) == -2, (i, x)


def test_types_on_the_cpu():
    """64-bit inputs are computed in 64 bits; whole numbers are refused."""
    torch.manual_seed(3)
    q, k, v = (torch.randn(2, 7, n, 8, dtype=torch.float64, requires_grad=True) for n in (4, 2, 2))
    n = torch.tensor([7, 3])
    assert torch.autograd.gradcheck(lambda *t: attention(*t, causal=True, lengths=n), (q, k, v))
    with pytest.raises(TypeError):
        attention(*(torch.ones(1, 2, 1, 8, dtype=torch.int32),) * 3)


def test_encoder_on_a_padded_batch():
    from tips_b200.models.bert import synthetic_mlm_batch, tiny_bert
    torch.manual_seed(0)
    model = tiny_bert(dtype=torch.float32, device="cpu")
    ids, pos, labels = synthetic_mlm_batch(3, 64, 1024, seed=1)
    n = torch.tensor([64, 20, 33])
    pos = pos % n[:, None]
    other = torch.where(torch.arange(64)[None] < n[:, None], ids, (ids + 7) % 1024)
    a, b = (model.loss(x, pos, labels, lengths=n) for x in (ids, other))
    assert torch.allclose(a, b, rtol=1e-5)
    assert not torch.allclose(a, model.loss(ids, pos, labels), rtol=1e-5)


def test_the_encoder_reports_launches_whose_waits_ran_out(monkeypatch):
    from tips_b200.models.bert import tiny_bert
    from tips_b200.ops import attention as a, linear
    model = tiny_bert(dtype=torch.float32, device="cpu")
    for gemm, att, message in ((0, 0, None), (0, 4, "attention"), (3, 0, "GEMM")):
        monkeypatch.setattr(linear, "gemm_status", lambda: gemm)
        monkeypatch.setattr(a, "attention_status", lambda: att)
        if message is None:
            model.check()
        else:
            with pytest.raises(RuntimeError, match=message):
                model.check()


def test_what_is_too_large_for_a_gpu_is_a_value_error():
    """Without a GPU: the checks look at a tensor's type, device and number of sequences only."""
    from types import SimpleNamespace

    from tips_b200.ops.attention import _check_attention

    def check(b=1, s=16, h=2, hk=2, d=64, scale=None):
        return _check_attention(SimpleNamespace(shape=(b, s), dtype=torch.bfloat16, device="cuda", is_cuda=True), s, h, hk, d, None, scale)

    for ok in (dict(), dict(b=65535), dict(h=1 << 17, hk=1 << 17), dict(s=1 << 25), dict(s=1 << 24, h=4), dict(b=0, s=1 << 26), dict(b=1 << 20, s=0),
               dict(scale=2.0 ** -149), dict(scale=2.3e38)):
        check(**ok)
    for bad in (dict(b=65536), dict(h=(1 << 17) + 1, hk=(1 << 17) + 1), dict(s=(1 << 25) + 1), dict(s=(1 << 24) + 1, h=4), dict(b=1 << 12, s=1 << 16, h=512, hk=512),
                dict(scale=1e-50), dict(scale=2.4e38)):
        with pytest.raises(ValueError):
            check(**bad)
