"""The attention kernels against the formula in 64 bits, with bounds that count each rounding (attention_util.reference)."""
import math

import pytest
import torch

from attention_util import check, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(b, s, h, hk, d, dtype, seed=0, amp=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    q, k, v, do = (torch.randn(b, s, n, d, generator=g, device=DEV).mul(amp).to(dtype) for n in (h, hk, hk, h))
    return q.requires_grad_(), k.requires_grad_(), v.requires_grad_(), do


def run(q, k, v, do, **kw):
    from tips_b200.ops.attention import attention
    y = attention(q, k, v, **kw)
    dq, dk, dv = torch.autograd.grad(y, (q, k, v), do)
    return {"out": y.detach(), "dq": dq, "dk": dk, "dv": dv}


def status():
    from tips_b200.ops.attention import attention_status
    return attention_status()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,s,h,hk,d", [
    (1, 1, 1, 1, 64), (2, 2, 2, 1, 8), (1, 17, 3, 1, 40), (1, 127, 2, 2, 64), (1, 128, 1, 1, 128), (2, 129, 4, 2, 96),
    (1, 255, 2, 2, 32), (1, 257, 2, 1, 128), (2, 300, 6, 3, 72), (1, 513, 2, 2, 64), (1, 640, 8, 1, 120), (3, 384, 2, 2, 16),
    (1, 1500, 2, 1, 64), (1, 1031, 2, 2, 128)])
def test_sizes(b, s, h, hk, d, causal):
    dtype = torch.bfloat16 if (s + d) % 3 else torch.float16
    q, k, v, do = make(b, s, h, hk, d, dtype, seed=s)
    check(run(q, k, v, do, causal=causal), *reference(q, k, v, do, causal))
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[0, 1, 333, 128], [200, 0, 0, 129], [127, 256, 257, 2], [-5, 1000, 64, 300]])
def test_padded_batches(lengths, causal, dtype):
    """Lengths of nothing, of one, at and around the tiles' borders and out of range; NaN and infinities in the padding."""
    q, k, v, do = make(4, 333, 4, 2, 64, dtype, seed=sum(lengths))
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32 if causal else torch.int64)
    want, bound = reference(q, k, v, do, causal, n)
    with torch.no_grad():
        for i, m in enumerate(lengths):
            m = max(0, min(333, m))
            for t, x in ((q, math.nan), (k, math.inf), (v, math.nan), (do, -math.inf)):
                t[i, m:] = x
    got = run(q, k, v, do, causal=causal, lengths=n)
    check(got, want, bound)
    for i, m in enumerate(lengths):
        for x in got.values():
            assert not x[i, max(0, min(333, m)):].any()  # exactly zero


def test_scale_and_large_scores():
    """Scores of some hundred: the running maximum carries the row."""
    q, k, v, do = make(2, 400, 2, 2, 64, torch.bfloat16, seed=3, amp=2.0)
    check(run(q, k, v, do, scale=0.5, causal=True), *reference(q, k, v, do, True, scale=0.5))


@pytest.mark.parametrize("of_do,of_v", [(1e-5, 1.0), (3e3, 1.0), (1.0, 500.0), (1e-4, 1e-3), (0.0, 1.0), (200.0, 200.0)])
@pytest.mark.parametrize("d", [64, 96])
def test_fp16_gradients_of_any_size(d, of_do, of_v):
    """Gradients near fp16's smallest numbers, and products far beyond its largest, on their way to results within its range; one
    of the heads that share a key head has far smaller gradients."""
    q, k, v, do = make(2, 300, 4, 2, d, torch.float16, seed=21)
    with torch.no_grad():
        v.mul_(of_v)
        do.mul_(of_do)
        do[:, :, 1] *= 2.0 ** -6
        k.mul_(min(1.0, 1.0 / (of_do * of_v + 1e-9)))  # results stay finite
        q.mul_(min(1.0, 1.0 / (of_do * of_v + 1e-9)))
    want, bound = reference(q, k, v, do)
    assert max(float(x.abs().max()) for x in want.values()) < 6e4
    check(run(q, k, v, do), want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("s,d", [(5, 64), (48, 40), (128, 128)])
def test_short_rows_lose_nothing_in_their_difference(s, d, causal, dtype):
    """Rows of up to 128 keys hold D and dS more exactly than in 16 bits.  What is left is the rounding of dQ and dK themselves, r = u
    sqrt(1/3 * 3/(8 ln 2)) = 0.425 u in the 2-norm (uniform over half a step, magnitudes spread evenly over an octave), and that of the
    forward pass's probabilities, which reaches D by O.  It moves D by sum_j dP_j eps_j P_j with eps of size r: of n keys of like weight P
    and dP of size a by r P a sqrt(n); dQ by that times sum_j P K_j, of size P sqrt(n) |K|, with P = 1 / n, against dQ's own P a sqrt(n)
    |K|: by r / sqrt(n).  With 5 keys both together make 0.466 u, and 0.49 u allows for the sample.  The rounding of dS alone would make
    it 0.63 u with 5 keys and 0.60 u with many."""
    q, k, v, do = make(8, s, 16, 8, d, dtype, seed=31)
    got = run(q, k, v, do, causal=causal)
    want, _ = reference(q, k, v, do, causal)
    u = torch.finfo(dtype).eps / 2
    for name in ("dq", "dk"):
        off = float((got[name].double() - want[name]).norm() / want[name].norm())
        assert off <= 0.49 * u, (name, off / u)


def test_rising_scores_rescale_the_output():
    """Every key tile raises the maximum of every row."""
    q, k, v, do = make(1, 700, 2, 1, 64, torch.bfloat16, seed=4)
    with torch.no_grad():
        q[..., 0] = 4.0
        k[..., 0] = torch.linspace(-40, 40, 700, device=DEV)[None, :, None].to(k.dtype)
    check(run(q, k, v, do), *reference(q, k, v, do))


def test_strides_orders_and_alignment():
    """[b, h, s, d] order, slices of wider tensors, rows that start on 4 bytes, a broadcast key head and a broadcast gradient."""
    b, s, h, d = 2, 200, 4, 64
    q, k, v, do = make(b, s, h, h, d, torch.bfloat16, seed=5)
    want, bound = reference(q, k, v, do)

    def leaf(t):
        return t.detach().requires_grad_()

    def other(t, kind):
        if kind == "heads first":
            return t.detach().transpose(1, 2).contiguous().transpose(1, 2)
        if kind == "batch last":
            return t.detach().permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)
        if kind == "wide":
            return torch.cat([t.detach(), t.detach()], 3)[..., :d]
        if kind == "odd start":
            return torch.cat([t.detach()[..., :2], t.detach()], 3)[..., 2:]
        return t.detach().transpose(1, 3).contiguous().transpose(1, 3)  # last axis not contiguous

    for kind in ("heads first", "batch last", "wide", "odd start", "columns"):
        check(run(*(leaf(other(t, kind)) for t in (q, k, v)), other(do, kind)), want, bound)
    one = k.detach()[:, :, :1]
    want, bound = reference(q, one.expand(b, s, h, d), v, do)
    got = run(leaf(q), leaf(one.expand(b, s, h, d)), leaf(v), do)
    check(got, want, bound)
    ones = torch.ones((), device=DEV, dtype=q.dtype).expand(b, s, h, d)
    check(run(leaf(q), leaf(k), leaf(v), ones), *reference(q, k, v, ones))


@pytest.mark.parametrize("h,hk,lengths", [(4, 4, None), (6, 2, [70, 190])])
def test_packed(h, hk, lengths):
    from tips_b200.ops.attention import packed_attention
    b, s, d = 2, 190, 32
    q, k, v, do = make(b, s, h, hk, d, torch.bfloat16, seed=6)
    n = None if lengths is None else torch.tensor(lengths, device=DEV)
    want, bound = reference(q, k, v, do, False, n)
    qkv = torch.cat([t.detach().reshape(b, s, -1) for t in (q, k, v)], 2).requires_grad_()
    y = packed_attention(qkv, h, kv_heads=hk, lengths=n)
    (g,) = torch.autograd.grad(y, qkv, do.reshape(b, s, -1))
    g = g.view(b, s, h + 2 * hk, d)
    check({"out": y.detach().view(b, s, h, d), "dq": g[:, :, :h], "dk": g[:, :, h:h + hk], "dv": g[:, :, h + hk:]}, want, bound)


def test_gradient_against_differences():
    """<dO, O(x + e w)> in 64 bits, by central differences, against the gradients' product with w."""
    q, k, v, do = make(1, 150, 4, 2, 40, torch.bfloat16, seed=8)
    got = run(q, k, v, do, causal=True)
    _, bound = reference(q, k, v, do, True)
    g = torch.Generator(device=DEV)
    g.manual_seed(9)
    e = 1e-4
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        w = torch.randn(t.shape, generator=g, device=DEV, dtype=torch.float64)
        vals = []
        for sign in (1, -1):
            args = [x.detach().double() + (sign * e * w if x is t else 0) for x in (q, k, v)]
            out, _ = reference(*args, do.double(), True, store=torch.bfloat16)
            vals.append(float((out["out"] * do.double()).sum()))
        slope = (vals[0] - vals[1]) / (2 * e)
        # e^2 times the third derivative is far below the bound's 2^-8
        assert abs(slope - float((got[name].double() * w).sum())) <= float((bound[name] * w.abs()).sum())


def test_the_same_bits_twice_on_other_streams_and_in_graphs():
    q, k, v, do = make(2, 500, 4, 2, 64, torch.bfloat16, seed=10)
    n = torch.tensor([500, 131], device=DEV)
    first = run(q, k, v, do, lengths=n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(q, k, v, do, lengths=n)
    torch.cuda.current_stream().wait_stream(side)
    for name in first:
        assert torch.equal(first[name], other[name]), name
    # two graphs with their own outputs; replayed on other inputs, then in turn
    from tips_b200.ops.attention import _attention_bwd, _attention_fwd, _view
    bufs = [t.detach().clone() for t in (q, k, v, do)]
    views = [_view(t) for t in bufs[:3]]
    shape = (2, 500, 4, 2, 64)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = _attention_fwd(bufs[0], shape, *views, n, 0.125, False)
            grads = [torch.empty_like(t) for t in bufs[:3]]
            _attention_bwd(bufs[3], shape, *views, out, lse, n, 0.125, False, *(_view(t) for t in grads))
        graphs.append((g, dict(zip(("out", "dq", "dk", "dv"), (out, *grads)))))
    for t, x in zip(bufs, make(2, 500, 4, 2, 64, torch.bfloat16, seed=11)):
        t.copy_(x)
    n.copy_(torch.tensor([60, 499], device=DEV))
    want = run(*(t.clone().requires_grad_() for t in bufs[:3]), bufs[3], lengths=n)
    for g, got in graphs + graphs[:1]:
        g.replay()
        for name in want:
            assert torch.equal(got[name], want[name]), name
    assert status() == 0


def test_infinities_in_valid_places_are_not_hidden():
    q, k, v, do = make(1, 200, 1, 1, 64, torch.bfloat16, seed=12)
    with torch.no_grad():
        v[0, 7, 0, 3] = math.inf
    got = run(q, k, v, do)
    assert not got["out"][..., 3].isfinite().any() and got["out"][..., 4].isfinite().all()
    assert not got["dq"].isfinite().all()


def test_scores_of_minus_infinity():
    """Keys whose scores are -inf, as many as a whole tile holds, do not count, wherever they stand."""
    from tips_b200.ops.attention import attention
    for first in (True, False):
        q, k, v, _ = make(2, 300, 4, 2, 64, torch.bfloat16, seed=13)
        with torch.no_grad():
            q[..., 0] = -1.0
            k[..., 0] = 0.5
            hidden = slice(0, 140) if first else slice(100, 300)
            k[:, hidden, :, 0] = math.inf
            got = attention(q, k, v)
            seen = slice(140, 300) if first else slice(0, 100)
            x = (q.double().transpose(1, 2) @ k[:, seen].double().transpose(1, 2).repeat_interleave(2, 1).mT) / 8
            p, vd = torch.softmax(x, -1), v[:, seen].double().transpose(1, 2).repeat_interleave(2, 1)
            want = (p @ vd).transpose(1, 2)
            # the probabilities and the output are rounded once each; 2^-14 for what is held in 32 bits
            bound = (2.0 ** -8 + 2.0 ** -14) * (p @ vd.abs()).transpose(1, 2) + 2.0 ** -8 * want.abs()
        assert ((got.double() - want).abs() <= bound).all()


def test_fp16_many_small_probabilities():
    """One key takes nearly all of every row's weight; thousands of others, each 2^-26 of it, make up the output."""
    from tips_b200.ops.attention import attention
    s, d = 8192, 64
    q, k, v = (torch.zeros(1, s, 1, d, device=DEV, dtype=torch.float16) for _ in range(3))
    q[..., 0] = 1.0
    k[:, 0, :, 0] = 18.0  # e^-18: 2^-25.97
    v[:, 1:] = 1000.0
    got = attention(q, k, v, scale=1.0).double()
    p = math.exp(-18.0)
    want = 1000.0 * (s - 1) * p / (1 + (s - 1) * p)
    # a probability held times 2^7 is off by fp16's smallest half step, 2^-25, at most; a half step of the output; 2^-14 for 32 bits
    assert float((got - want).abs().max()) <= 1000.0 * (s - 1) * 2.0 ** -32 + (2.0 ** -11 + 2.0 ** -14) * want


def test_offsets_beyond_32_bits():
    """Sequences of a batch that lie more than 2^31 elements apart, every tensor in one buffer of 4.3 GB."""
    b, s, h, d = 2, 150, 2, 64
    step = 2 ** 31 + 64
    buf = torch.zeros(step + 4 * s * h * d, device=DEV, dtype=torch.bfloat16)
    q, k, v, do = make(b, s, h, h, d, torch.bfloat16, seed=14)
    far = [buf.as_strided((b, s, h, d), (step, h * d, d, 1), i * s * h * d) for i in range(4)]
    for t, x in zip(far, (q, k, v, do)):
        t.copy_(x.detach())
    n = torch.tensor([150, 99], device=DEV)
    want = run(q, k, v, do, lengths=n)
    got = run(*(t.detach().requires_grad_() for t in far[:3]), far[3], lengths=n)
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_fp16_backward_in_a_graph():
    """The largest magnitudes that scale fp16's gradients are found anew in every replay."""
    from tips_b200.ops.attention import _attention_bwd, _attention_fwd, _view
    shape = (2, 300, 4, 2, 64)
    bufs = [t.detach().clone() for t in make(*shape, torch.float16, seed=15)]
    views = [_view(t) for t in bufs[:3]]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = _attention_fwd(bufs[0], shape, *views, None, 0.125, True)
        grads = [torch.empty_like(t) for t in bufs[:3]]
        _attention_bwd(bufs[3], shape, *views, out, lse, None, 0.125, True, *(_view(t) for t in grads))
    for amp in (100.0, 1e-3, 1.0):
        for t, x in zip(bufs, make(*shape, torch.float16, seed=16)):
            t.copy_(x.detach())
        bufs[3].mul_(amp)
        want = run(*(t.clone().requires_grad_() for t in bufs[:3]), bufs[3], causal=True)
        g.replay()
        for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            assert torch.equal(x, want[name]), (name, amp)


def test_refusals_on_a_gpu():
    from tips_b200.ops.attention import attention, packed_attention
    q, k, v, _ = make(1, 16, 2, 2, 64, torch.bfloat16)
    with pytest.raises(TypeError):
        attention(q.float(), k.float(), v.float())
    big = torch.zeros(1, 16, 2, 136, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention(big, big, big)
    with pytest.raises(ValueError):
        attention(big[..., :12], big[..., :12], big[..., :12])
    with pytest.raises(ValueError):
        attention(q, k, v, lengths=torch.tensor([16]))  # on the CPU
    with pytest.raises(TypeError):
        attention(q, k.cpu(), v)
    with pytest.raises(ValueError):
        packed_attention(torch.zeros(1, 16, 384, device=DEV, dtype=torch.bfloat16), 5, kv_heads=1, scale=1.0)
    # gradients of gradients are refused, not wrong
    y = attention(q, k, v)
    (g,) = torch.autograd.grad(y.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_empty_inputs():
    from tips_b200.ops.attention import attention
    for b, s in ((0, 5), (3, 0)):
        x = torch.zeros(b, s, 2, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        y = attention(x, x, x)
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape


def test_encoder_on_a_padded_batch():
    """What stands in the padding does not matter, and a full batch matches the unpadded path."""
    from tips_b200.models.bert import synthetic_mlm_batch, tiny_bert
    torch.manual_seed(0)
    model = tiny_bert()
    ids, pos, labels = (t.to(DEV) for t in synthetic_mlm_batch(3, 64, 1024, seed=1))
    n = torch.tensor([64, 20, 33], device=DEV)
    pos = pos % n[:, None]
    other = torch.where(torch.arange(64, device=DEV)[None] < n[:, None], ids, (ids + 7) % 1024)
    grads = []
    for x in (ids, other):
        model.zero_grad()
        loss = model.loss(x, pos, labels, lengths=n)
        loss.backward()
        grads.append([loss.detach()] + [p.grad.clone() for p in model.layers.parameters()])
    # dropped positions still pass the row-wise layers, whose weight gradients they reach with factors of exactly zero
    for a, b in zip(*grads):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=2 ** -8 * float(a.float().abs().max()))
    full = torch.full((3,), 64, device=DEV)
    a, b = model.encode(ids), model.encode(ids, full)
    assert (a.float() - b.float()).norm() <= 2 ** -5 * a.float().norm()


def test_the_status_waits_for_every_stream():
    """A launch that is still running, or to come, on a stream of its own is not reported as sound."""
    from tips_b200.ops.linear import gemm_status
    q, k, v, do = make(1, 64, 1, 1, 64, torch.bfloat16)
    run(q, k, v, do)
    torch.cuda.synchronize()
    for ask in (status, gemm_status):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.cuda._sleep(400_000_000)  # about a fifth of a second
            run(q, k, v, do)
        assert not side.query()
        assert ask() == 0 and side.query()


def test_the_most_sequences_of_a_launch():
    from tips_b200.ops.attention import attention, packed_attention
    q, k, v, do = make(65535, 3, 1, 1, 8, torch.bfloat16, seed=40)
    check(run(q, k, v, do, causal=True), *reference(q, k, v, do, True))
    assert status() == 0
    x = torch.zeros(65536, 3, 1, 8, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention(x, x, x)
    with pytest.raises(ValueError):
        packed_attention(x.expand(65536, 3, 3, 8).reshape(65536, 3, 24), 1, scale=1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 128), (6, 2, 80), (4, 1, 128), (3, 1, 96)])
@pytest.mark.parametrize("lengths", [[0, 1, 333, 128], [65, 256, 257, 191]])
def test_padded_batches_of_larger_heads(lengths, h, hk, d, causal, dtype):
    """Heads above 64 have a warp that clears what lies beyond a length, two sets of softmax warps, and outputs that are stored
    directly: lengths around units of 64 and tiles of 128, NaN and infinities in the padding."""
    q, k, v, do = make(4, 333, h, hk, d, dtype, seed=sum(lengths) + d)
    n = torch.tensor(lengths, device=DEV)
    want, bound = reference(q, k, v, do, causal, n)
    with torch.no_grad():
        for i, m in enumerate(lengths):
            for t, x in ((q, -math.inf), (k, math.nan), (v, math.inf), (do, math.nan)):
                t[i, m:] = x
    got = run(q, k, v, do, causal=causal, lengths=n)
    check(got, want, bound)
    for i, m in enumerate(lengths):
        for x in got.values():
            assert not x[i, m:].any()
    assert status() == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_pieces_follow_one_another(causal, d):
    """Several pieces of work per block, of one unit to many and some of none, most of them with rows to clear: what a block carries
    over from piece to piece (phases of its barriers, ring places, stores that are owed) does not depend on where a piece ends."""
    b, s, h, hk = 40, 700, 8, 2
    q, k, v, do = make(b, s, h, hk, d, torch.bfloat16, seed=50)
    g = torch.Generator()
    g.manual_seed(51)
    n = torch.randint(0, s + 1, (b,), generator=g)
    n[3], n[17], n[30] = 0, s, 1
    n = n.to(DEV)
    got = run(q, k, v, do, causal=causal, lengths=n)
    assert status() == 0
    for i in range(0, b, 8):  # in parts: the reference holds several [heads, s, s] matrices in 64 bits
        part = slice(i, i + 8)
        want, bound = reference(q[part], k[part], v[part], do[part], causal, n[part])
        check({name: x[part] for name, x in got.items()}, want, bound)


def test_scores_of_minus_infinity_at_a_large_scale():
    """What stands for the maximum of a row whose first keys' scores are -inf stays finite when it is scaled."""
    from tips_b200.ops.attention import attention
    q, k, v, _ = make(1, 300, 2, 2, 64, torch.bfloat16, seed=14)
    with torch.no_grad():
        q.mul_(2.0 ** -30)
        q[..., 0] = -1.0
        k[..., 0] = 0.0
        k[:, :140, :, 0] = math.inf
        got = attention(q, k, v, scale=2.0 ** 29)
        seen = slice(140, 300)
        x = (q.double().transpose(1, 2) @ k[:, seen].double().transpose(1, 2).mT) * 2.0 ** 29
        p, vd = torch.softmax(x, -1), v[:, seen].double().transpose(1, 2)
        want = (p @ vd).transpose(1, 2)
        # the probabilities and the output are rounded once each; 2^-14 for what is held in 32 bits
        bound = (2.0 ** -8 + 2.0 ** -14) * (p @ vd.abs()).transpose(1, 2) + 2.0 ** -8 * want.abs()
    assert ((got.double() - want).abs() <= bound).all()
