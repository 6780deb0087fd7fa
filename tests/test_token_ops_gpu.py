"""Rotary positions, norm of queries and keys, sliding-window attention: every kernel against the float64 oracle, with elementwise bounds
that follow from the arithmetic (oracle/ref_tokens.py), at the sizes, windows and layouts where such kernels go wrong."""
import math

import pytest
import torch

from oracle import ref_tokens as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0 ** -24}      # (fp16 results below 2^-14 round to a fixed step)


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def rnd(shape, seed, dev, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dev, dtype)


def within(got, want, bound, what, dtype):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.numel():
        return
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound - TINY[dtype]).max().item()
    worst = ((got - want).abs() / (bound + TINY[dtype])).max().item()
    assert over <= 0, f"{what}: {worst:.2f} of the bound"


def grid(D, H, W, prefix, dev, dtype=torch.int32):
    g = torch.stack(torch.meshgrid(torch.arange(D), torch.arange(H), torch.arange(W), indexing="ij"), -1).reshape(-1, 3)
    return torch.cat((torch.zeros(prefix, 3, dtype=torch.long), g)).to(dev, dtype)


# ------------------------------------------------------------------------------------------------ rotary
# (positions' type, heads, d, sections, interleaved): partial heads, an axis without pairs, one to four axes
ROT = [(torch.int32, 3, 64, (12, 10, 10), False), (torch.int64, 1, 128, (22, 21, 21), True), (torch.float32, 5, 32, (6, 5, 5), False),
       (torch.int32, 2, 96, (16, 0, 8), True), (torch.int32, 7, 96, (48,), False), (torch.int64, 2, 64, (4, 4, 4, 4), False)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", ROT)
def test_rotary_axes_and_its_gradient(dtype, case):
    """A turn of (a, b): cos, sin and both products in fp32 (together below 8 E of |a| + |b|), one rounding to the storage type."""
    from dose_prediction_amd import ops
    dev = _dev()
    kind, heads, d, sections, inter = case
    B, N, axes = 2, 37, len(sections)
    pos = torch.randint(-40, 4000, (B, N, axes), generator=torch.Generator().manual_seed(1)).to(dev, kind)
    if kind == torch.float32:
        pos = pos / 8
    x = rnd((B, N, heads * d + 32), 2, dev, dtype)[..., 16:16 + heads * d].requires_grad_()         # a slice of wider rows
    g = rnd((B, N, heads * d), 3, dev, dtype)
    y = ops.rotary_axes(x, heads, pos, sections, interleaved=inter)
    (gx,) = torch.autograd.grad(y, x, g)
    xr, gr = (t.detach().double().unflatten(-1, (heads, d)) for t in (x, g))
    u = R.half_step(dtype)
    want = R.rotary(xr, pos, sections, interleaved=inter)
    within(y.unflatten(-1, (heads, d)), want, u * want.abs() + 8 * R.E * R.pair_size(xr, inter), "y", dtype)
    back = R.rotary(gr, -pos.double(), sections, interleaved=inter)
    within(gx.unflatten(-1, (heads, d)), back, u * back.abs() + 8 * R.E * R.pair_size(gr, inter), "gx", dtype)


def test_rotary_far_positions_and_shared_tables():
    """Angles of far positions keep their fraction of a turn (2^40 positions: 64-bit reduction leaves 2^40 * 2^-53 of a radian), one table
    serves all sequences, an expanded input is read in place, and turning back returns the input."""
    from dose_prediction_amd import ops
    dev = _dev()
    B, N, heads, d = 3, 9, 2, 64
    pos = (torch.arange(N * 3).reshape(N, 3) + (1 << 40)).to(dev)
    x = rnd((1, N, heads * d), 4, dev).expand(B, N, heads * d)
    y = ops.rotary_axes(x, heads, pos, (12, 10, 10))
    xr = x.double().unflatten(-1, (heads, d))
    want = R.rotary(xr, pos, (12, 10, 10))
    within(y.unflatten(-1, (heads, d)), want, (8 * R.E + 2.0 ** -11) * R.pair_size(xr), "far", torch.float32)
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
    pos = pos - (1 << 40)
    there = ops.rotary_axes(x, heads, pos, (12, 10, 10))
    back = ops.rotary_axes(there, heads, -pos, (12, 10, 10))
    assert (back - x).abs().max().item() < 32 * R.E * 2 * x.abs().max().item()


# ------------------------------------------------------------------------------------------------ norm of queries and keys
def _norm_oracle(x, ws, heads, kv, pos, sections, inter, g):
    leaves = [x.detach().double().requires_grad_()] + [w.detach().double().requires_grad_() for w in ws]
    h = leaves[0].unflatten(-1, (heads + kv, -1))
    y = torch.cat((R.head_norm(h[:, :, :heads], leaves[1], leaves[2]), R.head_norm(h[:, :, heads:], leaves[3], leaves[4])), 2)
    if pos is not None:
        y = R.rotary(y, pos, sections, interleaved=inter)
    y = y.flatten(-2)
    return y.detach(), torch.autograd.grad(y, leaves, g.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,N,heads,kv,d,inter,rot", [(1, 1, 1, 1, 32, False, True), (2, 41, 6, 2, 64, True, True), (1, 700, 3, 3, 96, False, True),
                                                      (3, 175, 2, 1, 128, True, False), (1, 2500, 4, 4, 128, False, True)])
def test_qk_norm_rotary(dtype, B, N, heads, kv, d, inter, rot):
    """Statistics in fp32 over d values: |h| <= sqrt(d), its error below 8 E (1 + |mean| rstd) sqrt(d) -- inputs here have |mean| rstd <= 2 --,
    the turn adds its own; the gradient of a normalised row sums d products, 3 of them: 4 d E of the largest terms; weight gradients are
    sums over R rows, fp32 per thread and 64 bits behind that, of terms whose own error is as above."""
    from dose_prediction_amd import ops
    dev = _dev()
    x = (rnd((B, N, (heads + 2 * kv) * d), 5, dev) + 1.0).to(dtype)[..., :(heads + kv) * d].requires_grad_()
    ws = [(rnd((d,), 6 + i, dev, scale=0.2) + (i + 1) % 2).requires_grad_() for i in range(4)]
    g = rnd((B, N, (heads + kv) * d), 10, dev, dtype)
    pos = grid(1, 1, N, 0, dev) + 3 if rot else None
    sec = ((d // 2 - 2 * (d // 6)), d // 6, d // 6) if rot else None
    y = ops.qk_norm_rotary(x, heads, kv, *ws, positions=pos, sections=sec, interleaved=inter)
    got = torch.autograd.grad(y, [x, *ws], g)
    want, grads = _norm_oracle(x, ws, heads, kv, pos, sec, inter, g)
    u, wmax = R.half_step(dtype), max(w.abs().max().item() for w in ws)
    eh = 8 * R.E * 3 * math.sqrt(d)
    within(y, want, u * want.abs() + 2 * (eh * wmax + 8 * R.E * (math.sqrt(d) * wmax + wmax)), "y", dtype)
    rstd = (x.detach().double().unflatten(-1, (heads + kv, d)).var(-1, unbiased=False) + 1e-5).rsqrt().max().item()
    gmax = 2 * g.abs().max().item()
    within(got[0], grads[0], u * grads[0].abs() + 4 * rstd * gmax * wmax * (1 + d ** 0.5) * (eh + d * R.E), "gx", dtype)
    for i, name in enumerate(("q_weight", "q_bias", "k_weight", "k_bias")):
        rows = B * N * (heads if i < 2 else kv)
        per = (eh + 16 * R.E * math.sqrt(d)) * gmax       # one term's error; a thread adds at most rows / 64 of them in fp32, errors of rows add up
        within(got[1 + i], grads[1 + i], torch.full_like(grads[1 + i], rows * per), name, torch.float32)
        assert ((got[1 + i].double() - grads[1 + i]).norm() / grads[1 + i].norm()).item() < 1e-4
    again = torch.autograd.grad(ops.qk_norm_rotary(x, heads, kv, *ws, positions=pos, sections=sec, interleaved=inter), [x, *ws], g)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


# ------------------------------------------------------------------------------------------------ attention
# name: (B, Nq, Nk, heads, kv, d, left, right, sinks, q_start, lengths)
WIN = {
    "one_token": (1, 1, 1, 1, 1, 64, None, None, 0, 0, None),
    "itself_only": (2, 7, 7, 3, 3, 64, 0, 0, 0, 0, None),
    "small_window_sinks": (1, 33, 33, 4, 4, 32, 5, 3, 2, 0, None),
    "look_back_shared_heads": (2, 129, 129, 6, 2, 96, None, 0, 0, 0, None),
    "look_ahead": (1, 70, 70, 2, 1, 128, 0, None, 0, 0, None),
    "ragged": (4, 257, 257, 2, 2, 128, 100, 20, 4, 0, (257, 0, 100, 1)),
    "ragged_shared": (3, 95, 95, 6, 2, 64, 31, 32, 1, 0, (95, 33, 64)),
    "everything": (1, 200, 200, 2, 2, 96, None, None, 9, 0, None),
    "sinks_over_tiles": (1, 3000, 3000, 2, 1, 64, 16, 16, 200, 0, None),
    "more_sinks_than_keys": (1, 90, 90, 2, 2, 64, 3, 3, 1000, 0, None),
    "last_queries": (2, 5, 300, 4, 2, 64, 64, 0, 3, 295, None),
    "queries_outside": (2, 40, 50, 2, 2, 64, 8, 8, 1, (-10, 45), (50, 47)),
    "more_queries_than_keys": (1, 120, 30, 2, 2, 32, 10, 10, 0, 0, None),
    "wide_64": (2, 1100, 1100, 16, 16, 64, 150, 77, 3, 0, (1100, 900)),
    "wide_128": (1, 1033, 1033, 32, 32, 128, 200, 0, 70, 0, None),
    "wide_96_shared": (4, 700, 700, 36, 12, 96, 64, 64, 0, 0, (700, 650, 699, 1)),
    "few_key_tiles": (1, 600, 600, 6, 2, 64, None, 0, 0, 0, None),
    "few_key_tiles_sinks": (2, 700, 700, 6, 1, 96, 300, 40, 50, 0, (700, 333)),
    "few_key_tiles_outside": (1, 1500, 1300, 3, 1, 128, 500, None, 40, -100, (1250,)),
    "wide_32": (8, 260, 260, 16, 16, 32, None, 0, 0, 0, None),
}


def _win_inputs(name, dtype, dev, seed=20, scale=1.0):
    B, Nq, Nk, heads, kv, d, left, right, sinks, start, lengths = WIN[name]
    q, k, v = rnd((B, Nq, heads, d), seed, dev, dtype, scale), rnd((B, Nk, kv, d), seed + 1, dev, dtype, scale), rnd((B, Nk, kv, d), seed + 2, dev, dtype)
    g = rnd((B, Nq, heads, d), seed + 3, dev, dtype)
    as_t = lambda s: torch.tensor(s, dtype=torch.int32, device=dev) if isinstance(s, tuple) else s  # noqa: E731
    return [t.requires_grad_() for t in (q, k, v)], g, dict(left=left, right=right, sinks=sinks), as_t(start), as_t(lengths)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(WIN))
def test_window_attention_forward_and_backward(name, dtype):
    from dose_prediction_amd import ops
    dev = _dev()
    (q, k, v), g, win, start, lengths = _win_inputs(name, dtype, dev)
    out = ops.window_attention(q, k, v, q_start=start, lengths=lengths, **win)
    grads = torch.autograd.grad(out, (q, k, v), g)
    want = R.window(q.detach(), k.detach(), v.detach(), g, start=start, lengths=lengths, dtype=dtype, **win)
    for what, got, (val, bound) in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), want):
        within(got, val, bound, what, dtype)
    again = ops.window_attention(q, k, v, q_start=start, lengths=lengths, **win)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(again, (q, k, v), g)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d,Nq", [(12, 4, 64, 1), (2, 2, 128, 1), (8, 1, 32, 4), (3, 3, 96, 2)])
def test_window_attention_few_queries_over_long_rows(dtype, heads, kv, d, Nq):
    """The form for single tokens: the keys are dealt to many blocks and joined; every sequence has its own length, one of them none."""
    from dose_prediction_amd import ops
    dev = _dev()
    B, Nk = 3, 5003
    q, k, v = rnd((B, Nq, heads, d), 30, dev, dtype), rnd((B, Nk, kv, d), 31, dev, dtype), rnd((B, Nk, kv, d), 32, dev, dtype)
    lengths = torch.tensor([5003, 0, 2049], dtype=torch.int32, device=dev)
    assert ops._window_ws(B, heads, kv, Nq, Nk, d, (-1, 0, 0), 0, dev) is not None
    for left in (None, 700):
        out = ops.window_attention(q, k, v, left=left, right=0, sinks=5, q_start=lengths - Nq, lengths=lengths)
        ((val, bound),) = R.window(q, k, v, left=left, right=0, sinks=5, start=lengths - Nq, lengths=lengths, dtype=dtype)
        within(out, val, bound, f"left={left}", dtype)


@pytest.mark.parametrize("name", ["small_window_sinks", "ragged", "wide_64"])
def test_window_attention_strides(name):
    """Slices of a packed projection, head-major tensors and a view at an odd offset (copied) give the bits of dense operands, and gradients
    arrive at the leaves behind the views; a gradient that is itself a view is read with its strides."""
    from dose_prediction_amd import ops
    dev = _dev()
    (q, k, v), g, win, start, lengths = _win_inputs(name, torch.bfloat16, dev)
    out = ops.window_attention(q, k, v, q_start=start, lengths=lengths, **win)
    grads = torch.autograd.grad(out, (q, k, v), g)
    B, N, heads, d = q.shape
    packed = torch.cat([t.detach().flatten(-2) for t in (q, k, v)], -1).requires_grad_()
    views = packed.unflatten(-1, (3 * heads, d)).split(heads, 2)
    major = [t.detach().transpose(1, 2).contiguous().requires_grad_() for t in (q, k, v)]
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)[1:].view(t.shape).copy_(t.detach()).requires_grad_() for t in (q, k, v)]
    gt = g.transpose(1, 2).contiguous().transpose(1, 2)
    o1 = ops.window_attention(*views, q_start=start, lengths=lengths, **win)
    o2 = ops.window_attention(*(t.transpose(1, 2) for t in major), q_start=start, lengths=lengths, **win)
    o3 = ops.window_attention(*odd, q_start=start, lengths=lengths, **win)
    assert torch.equal(out, o1) and torch.equal(out, o2) and torch.equal(out, o3)
    (gp,) = torch.autograd.grad(o1, packed, gt)
    assert torch.equal(gp, torch.cat([t.flatten(-2) for t in grads], -1))
    assert all(torch.equal(a, b.transpose(1, 2)) for a, b in zip(grads, torch.autograd.grad(o2, major, gt)))
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(o3, odd, g)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["ragged", "ragged_shared", "wide_64", "queries_outside"])
def test_padding_may_hold_anything(name, dtype):
    """NaN and infinities outside the sequences -- queries, keys, values and the incoming gradient -- change no bit; the padding's own rows and
    gradients are zero."""
    from dose_prediction_amd import ops
    dev = _dev()
    (q, k, v), g, win, start, lengths = _win_inputs(name, dtype, dev)
    ref = ops.window_attention(q, k, v, q_start=start, lengths=lengths, **win)
    grads = torch.autograd.grad(ref, (q, k, v), g)
    B, Nq, Nk = q.shape[0], q.shape[1], k.shape[1]
    pos = torch.as_tensor(start, device=dev).reshape(-1, 1).expand(B, 1) + torch.arange(Nq, device=dev)
    padq = ((pos < 0) | (pos >= lengths[:, None]))[..., None, None]
    padk = (torch.arange(Nk, device=dev) >= lengths[:, None])[..., None, None]
    assert padq.any()
    for bad in (math.nan, math.inf, -math.inf):
        q2, g2 = (t.detach().masked_fill(padq, bad).requires_grad_() for t in (q, g))
        k2, v2 = (t.detach().masked_fill(padk, bad).requires_grad_() for t in (k, v))
        out = ops.window_attention(q2, k2, v2, q_start=start, lengths=lengths, **win)
        got = torch.autograd.grad(out, (q2, k2, v2), g2.detach())
        assert torch.equal(out, ref) and all(torch.equal(a, b) for a, b in zip(got, grads))
    assert not ref.masked_select(padq).any() and not grads[0].masked_select(padq).any()
    assert not grads[1].masked_select(padk).any() and not grads[2].masked_select(padk).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_scores_and_scale(dtype):
    """Scores of several hundred: a softmax that is one key, a maximum that moves from tile to tile; a scale of its own."""
    from dose_prediction_amd import ops
    dev = _dev()
    (q, k, v), g, win, start, lengths = _win_inputs("ragged_shared", dtype, dev, seed=40)
    q2 = (q.detach() * 24).requires_grad_()
    k2 = (k.detach() * torch.linspace(0.1, 2, k.shape[1], device=dev).view(1, -1, 1, 1).to(dtype)).requires_grad_()
    for scale in (None, 0.03125):
        out = ops.window_attention(q2, k2, v, q_start=start, lengths=lengths, scale=scale, **win)
        grads = torch.autograd.grad(out, (q2, k2, v), g)
        want = R.window(q2.detach(), k2.detach(), v.detach(), g, start=start, lengths=lengths, scale=scale, dtype=dtype, **win)
        for what, got, (val, bound) in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), want):
            within(got, val, bound, what, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("step", [0.02, 0.4, 5.0])
def test_rising_scores(dtype, step):
    """Every key scores higher than the one before it, a window at a time: the running maximum creeps, steps and jumps, P passes 1 in between."""
    from dose_prediction_amd import ops
    dev = _dev()
    B, N, heads, d = 2, 300, 2, 64
    q = rnd((B, N, heads, d), 41, dev, scale=0.1)
    q[..., 0] = 8.0
    k = rnd((B, N, heads, d), 42, dev, scale=0.1)
    k[..., 0] = (step * torch.arange(N, device=dev) - step * 150).view(1, N, 1)
    q, k, v, g = (t.to(dtype) for t in (q, k, rnd((B, N, heads, d), 43, dev), rnd((B, N, heads, d), 44, dev)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    for win in (dict(), dict(left=70, right=40, sinks=3), dict(right=0)):
        out = ops.window_attention(*leaves, **win)
        grads = torch.autograd.grad(out, leaves, g)
        want = R.window(q.detach(), k.detach(), v.detach(), g, dtype=dtype, **win)
        for what, got, (val, bound) in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), want):
            within(got, val, bound, what, dtype)


def test_lengths_and_starts_past_32_bits():
    from dose_prediction_amd import ops
    dev = _dev()
    q, k, v = (rnd((3, 40, 2, 64), 45 + i, dev) for i in range(3))
    big = torch.tensor([(1 << 32) + 3, 1 << 40, -(1 << 35)], device=dev)
    got = ops.window_attention(q, k, v, left=9, lengths=big)
    assert torch.equal(got, ops.window_attention(q, k, v, left=9, lengths=torch.tensor([40, 40, 0], device=dev)))
    assert ops.window_attention(q, k, v, left=9, q_start=big).abs().max().item() == 0


def test_gradient_against_differences():
    """Directional derivative of the fp32 kernels: central differences with h = 2^-6 are off by h^2 times the third derivative (scores change by
    at most ~0.3 here: below 2e-3 of the terms' size) and by 2 E |f| / h."""
    from dose_prediction_amd import ops
    dev = _dev()
    (q, k, v), g, win, start, lengths = _win_inputs("small_window_sinks", torch.float32, dev, seed=50)
    f = lambda a, b, c: (ops.window_attention(a, b, c, **win) * g).double().sum().item()  # noqa: E731
    grads = torch.autograd.grad((ops.window_attention(q, k, v, **win) * g).sum(), (q, k, v))
    h = 2.0 ** -6
    for i, (t, gt) in enumerate(zip((q, k, v), grads)):
        dirn = rnd(tuple(t.shape), 60 + i, dev)
        plus, minus = [x.detach() for x in (q, k, v)], [x.detach() for x in (q, k, v)]
        plus[i], minus[i] = t.detach() + h * dirn, t.detach() - h * dirn
        diff, size = (f(*plus) - f(*minus)) / (2 * h), (gt.double().abs() * dirn.double().abs()).sum().item()
        assert abs(diff - (gt.double() * dirn.double()).sum().item()) < 2e-3 * size


def test_empty_sizes():
    from dose_prediction_amd import ops
    dev = _dev()
    for B, Nq, Nk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        q, k, v = (torch.randn(B, n, 2, 64, device=dev, requires_grad=True) for n in (Nq, Nk, Nk))
        out = ops.window_attention(q, k, v, left=2, right=2, sinks=1)
        grads = torch.autograd.grad(out.sum(), (q, k, v))
        assert out.shape == q.shape and not out.any() and all(x.shape == y.shape and not x.any() for x, y in zip(grads, (q, k, v)))
    x = torch.randn(2, 0, 4 * 64, device=dev, requires_grad=True)
    pos = torch.zeros(0, 3, dtype=torch.int32, device=dev)
    w = [torch.ones(64, device=dev, requires_grad=True) for _ in range(4)]
    y = ops.qk_norm_rotary(x, 2, 2, *w, positions=pos, sections=(12, 10, 10))
    grads = torch.autograd.grad(y.sum(), [x, *w])
    assert y.shape == x.shape and all(not t.any() for t in grads[1:])
    assert ops.rotary_axes(x, 4, pos, (12, 10, 10)).shape == x.shape


def test_offsets_past_32_bits():
    """Keys and values whose last rows lie more than 2^31 elements behind their first."""
    from dose_prediction_amd import ops
    dev = _dev()
    Nk, step, d = 33000, 1 << 16, 64
    base = torch.empty(Nk * step + d, dtype=torch.bfloat16, device=dev)
    k, v = (base[o:].as_strided((1, Nk, 1, d), (0, step, d, 1)) for o in (0, 64 * d))
    kd, vd = rnd((1, Nk, 1, d), 70, dev, torch.bfloat16), rnd((1, Nk, 1, d), 71, dev, torch.bfloat16)
    k.copy_(kd)
    v = base[64 * d:].as_strided((1, Nk - 1, 1, d), (0, step, d, 1))
    k = k[:, :Nk - 1]
    v.copy_(vd[:, :Nk - 1])
    q = rnd((1, 3, 1, d), 72, dev, torch.bfloat16)
    win = dict(left=None, right=0, q_start=Nk - 4)
    assert torch.equal(ops.window_attention(q, k, v, **win), ops.window_attention(q, kd[:, :Nk - 1].contiguous(), vd[:, :Nk - 1].contiguous(), **win))


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d,D,H,W,norm,inter", [(6, 6, 128, 4, 4, 5, True, False), (12, 4, 64, 3, 5, 7, False, True), (4, 2, 96, 2, 9, 9, True, True)])
def test_block_equals_its_parts(dtype, heads, kv, d, D, H, W, norm, inter):
    """window_attention_qkv runs the kernels of its parts: the same bits forward; backward the same in fp32, and in 16 bits apart by the one
    rounding of dq and dk that it saves (a turn passes it on as u (|a| + |b|); behind a norm: 4 rstd |w| times that, summed in its means)."""
    from dose_prediction_amd import ops
    dev = _dev()
    B, N = 2, 1 + D * H * W
    pos, sec = grid(D, H, W, 1, dev), (d // 2 - 2 * (d // 6), d // 6, d // 6)
    qkv = rnd((B, N, (heads + 2 * kv) * d), 80, dev, dtype).requires_grad_()
    ws = [(rnd((d,), 81 + i, dev, scale=0.2) + (i + 1) % 2).requires_grad_() for i in range(4)] if norm else None
    g = rnd((B, N, heads * d), 86, dev, dtype)
    win = dict(left=20, right=13, sinks=1, lengths=torch.tensor([N, N - 17], device=dev))
    one = ops.window_attention_qkv(qkv, heads, kv, norm=ws, positions=pos, sections=sec, interleaved=inter, **win)
    qk = qkv[..., :(heads + kv) * d]
    if norm:
        qk = ops.qk_norm_rotary(qk, heads, kv, *ws, positions=pos, sections=sec, interleaved=inter)
    else:
        qk = ops.rotary_axes(qk, heads + kv, pos, sec, interleaved=inter)
    q, k = qk.unflatten(-1, (heads + kv, d)).split((heads, kv), 2)
    q.retain_grad(), k.retain_grad()
    two = ops.window_attention(q, k, qkv[..., (heads + kv) * d:].unflatten(-1, (kv, d)), **win).flatten(-2)
    assert torch.equal(one, two)
    leaves = [qkv] + (ws or [])
    a = torch.autograd.grad(one, leaves, g)
    b = torch.autograd.grad(two, leaves, g)
    if dtype == torch.float32:
        assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1:], b[1:]))
        return
    u = R.half_step(dtype)
    # in the 2-norm: roundings of dq, dk and of the result, each at most u of the vector; a norm's backward map shortens (h and the mean taken
    # out) what it scales by rstd |w|, whose spread over heads and channels is below 4 here
    cut = (heads + kv) * d
    assert torch.equal(a[0][..., cut:], b[0][..., cut:])
    far = (a[0].double() - b[0].double())[..., :cut].norm() / b[0].double()[..., :cut].norm()
    assert far.item() <= u * (3 if not norm else 2 + 4)


def test_block_without_extras_equals_full_attention():
    """No window, norm or positions: the framework's attention() to the rounding of either (both within the oracle's bound)."""
    from dose_prediction_amd import ops
    dev = _dev()
    B, N, heads, d = 2, 150, 3, 128
    qkv = rnd((B, N, 3 * heads * d), 90, dev, torch.bfloat16)
    q, k, v = qkv.unflatten(-1, (3 * heads, d)).split(heads, 2)
    ((val, bound),) = R.window(q, k, v, dtype=torch.bfloat16)
    within(ops.attention(qkv, heads).unflatten(-1, (heads, d)), val, bound, "attention", torch.bfloat16)
    within(ops.window_attention_qkv(qkv, heads).unflatten(-1, (heads, d)), val, bound, "window_attention_qkv", torch.bfloat16)


def test_other_stream_and_captured_graph():
    """The launches go to the caller's stream, and a captured forward + backward replays with fresh inputs: every replay against the eager
    result, with eager work of the same operators in between."""
    from dose_prediction_amd import ops
    dev = _dev()
    heads, d, N = 4, 64, 1 + 6 * 6 * 6
    pos = grid(6, 6, 6, 1, dev)
    ws = [(rnd((d,), 101 + i, dev, scale=0.2) + (i + 1) % 2).requires_grad_() for i in range(4)]
    x = rnd((2, N, 3 * heads * d), 100, dev, torch.bfloat16).requires_grad_()
    g = rnd((2, N, heads * d), 106, dev, torch.bfloat16)

    def step():
        y = ops.window_attention_qkv(x, heads, left=30, right=30, sinks=1, norm=ws, positions=pos, sections=(12, 10, 10))
        return (y.detach(), *torch.autograd.grad(y, [x, *ws], g))
    side = torch.cuda.Stream()
    want = [t.clone() for t in step()]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(rnd(tuple(x.shape), 110 + i, dev, torch.bfloat16))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_calls_without_a_gradient():
    """No graph where none is asked for, the same bits as with one; a leaf that asks for a gradient gets one whatever the others do."""
    from dose_prediction_amd import ops
    dev = _dev()
    heads, d, N = 2, 64, 65
    pos = grid(4, 4, 4, 1, dev)
    x = rnd((2, N, 3 * heads * d), 120, dev, torch.bfloat16)
    ws = [rnd((d,), 121 + i, dev, scale=0.2) + (i + 1) % 2 for i in range(4)]
    q, k, v = x.unflatten(-1, (3 * heads, d)).split(heads, 2)
    rot = dict(positions=pos, sections=(12, 10, 10))
    calls = [(lambda: ops.rotary_axes(x, 3 * heads, **rot), [x]), (lambda: ops.qk_norm_rotary(x, heads, 2 * heads, *ws, **rot), [x, *ws]),
             (lambda: ops.window_attention(q, k, v, left=9), [q, k, v]), (lambda: ops.window_attention_qkv(x, heads, left=9, norm=ws, **rot), [x, *ws])]
    for call, leaves in calls:
        plain = call()
        assert not plain.requires_grad
        for leaf in leaves:
            leaf.requires_grad_()
            y = call()
            assert y.requires_grad and torch.equal(y, plain)
            (g,) = torch.autograd.grad(y.float().square().sum(), leaf)
            assert g.shape == leaf.shape and torch.isfinite(g).all()
            with torch.no_grad():
                z = call()
            assert not z.requires_grad and torch.equal(z, plain)
            leaf.requires_grad_(False)


def test_refused_on_the_gpu():
    from dose_prediction_amd import ops, _lib
    dev = _dev()
    q = torch.zeros(2, 4, 2, 64, device=dev)
    with pytest.raises(_lib.DoseHipError):
        ops.window_attention(q, q, q, lengths=torch.tensor([4, 4]))                  # lengths on the host
    with pytest.raises(TypeError):
        ops.window_attention(q, q.half(), q.half())
    with pytest.raises(_lib.DoseHipError):
        ops.rotary_axes(q.flatten(-2), 2, torch.zeros(4, 1, dtype=torch.int32), (4,))
