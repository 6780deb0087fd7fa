"""Token operators on the GPU: what their documentation promises of calls at its edges -- padding behind the norm and the rotation, tensors whose
outer strides mean nothing, recorded programs, gradients of gradients, the wide kernels behind the packed projection."""
import math

import pytest
import torch

from oracle import ref_tokens as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def rnd(shape, seed, dev, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dev, dtype)


def norms(d, seed, dev):
    return [(rnd((d,), seed + i, dev, scale=0.2) + (i + 1) % 2).requires_grad_() for i in range(4)]


# ------------------------------------------------------------------------------------------------ padding of a packed projection
# (heads, kv, d, interleaved, norm, rotary)
PACKED = [(4, 4, 64, False, True, True), (6, 2, 128, True, True, False), (4, 2, 96, True, False, True), (3, 3, 32, False, True, True)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", PACKED)
def test_packed_padding_may_hold_anything(dtype, case):
    """Rows outside the sequences -- the projection, the incoming gradient, the positions -- hold NaN or infinities: the same bits everywhere
    else, the norm's gradients among them, and zeros for their own gradient.  One sequence is empty, one is longer than the rows."""
    from dose_prediction_amd import ops
    dev = _dev()
    heads, kv, d, inter, norm, rot = case
    B, N = 4, 67
    lengths = torch.tensor([N, 0, 30, N + 5], dtype=torch.int32, device=dev)
    pad = torch.arange(N, device=dev) >= lengths[:, None]
    pos = torch.randint(0, 900, (B, N, 3), generator=torch.Generator().manual_seed(1)).to(dev, torch.float32)
    x, g = rnd((B, N, (heads + 2 * kv) * d), 2, dev, dtype), rnd((B, N, heads * d), 3, dev, dtype)
    ws = norms(d, 4, dev) if norm else []

    def step(x, g, pos):
        x = x.clone().requires_grad_()
        extra = dict(positions=pos, sections=(d // 2 - 2 * (d // 6), d // 6, d // 6), interleaved=inter) if rot else {}
        y = ops.window_attention_qkv(x, heads, kv, left=20, right=13, sinks=2, lengths=lengths, norm=ws or None, **extra)
        return (y.detach(), *torch.autograd.grad(y, [x, *ws], g))
    want = step(x, g, pos)
    for t in want:
        assert torch.isfinite(t).all()
    assert not want[0][pad].any() and not want[1][pad].any()
    for bad in (math.nan, math.inf, -math.inf):
        got = step(*(t.masked_fill(pad[..., None], bad) for t in (x, g, pos)))
        for name, a, b in zip(("out", "dqkv", "q_weight", "q_bias", "k_weight", "k_bias"), got, want):
            assert torch.equal(a, b), (name, bad)


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_padding_of_zeros_without_eps(dtype):
    """eps = 0 and a zero row behind the sequence: its variance is zero, its gradients are still none."""
    from dose_prediction_amd import ops
    dev = _dev()
    heads, d, N = 2, 64, 40
    lengths = torch.tensor([25, 40], dtype=torch.int32, device=dev)
    x = rnd((2, N, 3 * heads * d), 10, dev, dtype)
    x[0, 25:] = 0
    x.requires_grad_()
    ws = norms(d, 11, dev)
    y = ops.window_attention_qkv(x, heads, left=9, norm=ws, eps=0.0, lengths=lengths)
    grads = torch.autograd.grad(y, [x, *ws], rnd((2, N, heads * d), 15, dev, dtype))
    assert all(torch.isfinite(t).all() for t in (y, *grads)) and not grads[0][0, 25:].any()
    assert all(t.any() for t in grads)


# ------------------------------------------------------------------------------------------------ recorded programs
def _calls(dev, dtype=torch.bfloat16, N=65, heads=2, d=64):
    """(name, call of one tensor, that tensor): every operator as a function of the packed projection."""
    from dose_prediction_amd import ops
    x = rnd((2, N, 3 * heads * d), 20, dev, dtype)
    pos = torch.arange(3 * N, device=dev).reshape(N, 3)
    ws = [w.detach() for w in norms(d, 21, dev)]
    rot = dict(positions=pos, sections=(12, 10, 10))
    n = torch.tensor([N, 40], device=dev)

    def parts(t):
        return t.unflatten(-1, (3 * heads, d)).split(heads, 2)
    return [("rotary_axes", lambda t: ops.rotary_axes(t, 3 * heads, **rot), x),
            ("qk_norm_rotary", lambda t: ops.qk_norm_rotary(t, heads, 2 * heads, *ws, **rot), x),
            ("window_attention", lambda t: ops.window_attention(*parts(t), left=9, sinks=1, lengths=n), x),
            ("window_attention_qkv", lambda t: ops.window_attention_qkv(t, heads, left=9, norm=ws, lengths=n, **rot), x)]


@pytest.mark.filterwarnings("ignore")
def test_traced_programs_launch_the_kernels():
    """A recorded call computes on the inputs of the replay, where a gradient is asked for and where none is."""
    dev = _dev()
    for name, call, x in _calls(dev):
        traced = torch.jit.trace(call, (x,), check_trace=False)
        for i in range(3):
            y = rnd(tuple(x.shape), 30 + i, dev, x.dtype)
            want = call(y)
            assert torch.equal(traced(y), want), (name, i)
            with torch.no_grad():
                assert torch.equal(traced(y), want), (name, i)


@pytest.mark.filterwarnings("ignore")
def test_traced_transformer():
    """A transformer with a window, normed queries and keys and rotary positions, recorded for inference."""
    from dose_prediction_amd import blocks
    dev = _dev()
    torch.manual_seed(0)
    net = blocks.TransformerBlock(128, 256, 2, attention=dict(window=7, sinks=1, qk_norm=True, rotary=(12, 10, 10))).to(dev).eval()
    pos = torch.arange(3 * 40, device=dev, dtype=torch.int32).reshape(40, 3)
    x = [rnd((2, 40, 128), 40 + i, dev) for i in range(3)]
    with torch.no_grad():
        traced = torch.jit.trace(net, (x[0], pos), check_trace=False)
        for t in x:
            assert torch.equal(traced(t, pos), net(t, pos))


# ------------------------------------------------------------------------------------------------ strides of dimensions of one
def _odd_outer(t):
    """The same values in a view whose dimensions of one have odd strides (its rows are where they were)."""
    st = [s if n > 1 else 12345 + 2 * i for i, (n, s) in enumerate(zip(t.shape[:-1], t.stride()))]
    return t.as_strided(t.shape, (*st, 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,heads", [(1, 2), (33, 1), (33, 2)])
def test_strides_of_single_dimensions_do_not_matter(dtype, N, heads):
    from dose_prediction_amd import ops
    dev = _dev()
    d = 64
    pos = torch.arange(3 * N, device=dev).reshape(N, 3)
    ws = norms(d, 51, dev)
    rot = dict(positions=pos, sections=(12, 10, 10))
    x, g = rnd((1, N, 3 * heads * d), 50, dev, dtype), rnd((1, N, heads * d), 55, dev, dtype)
    g3 = rnd((1, N, 3 * heads * d), 56, dev, dtype)
    q, k, v = (t.contiguous() for t in x.unflatten(-1, (3 * heads, d)).split(heads, 2))
    g4 = g.unflatten(-1, (heads, d))
    calls = [(lambda a: ops.rotary_axes(a, 3 * heads, **rot), (x,), g3), (lambda a: ops.qk_norm_rotary(a, heads, 2 * heads, *ws, **rot), (x,), g3),
             (lambda a, b, c: ops.window_attention(a, b, c, left=5), (q, k, v), g4),
             (lambda a: ops.window_attention_qkv(a, heads, left=5, norm=ws, **rot), (x,), g)]
    for call, args, grad in calls:
        plain = [t.clone().requires_grad_() for t in args]
        odd = [_odd_outer(t.clone()).requires_grad_() for t in args]
        assert all(t.is_contiguous() for t in odd) and any(s % 2 for t in odd for s in t.stride()[:-1])
        want, got = call(*plain), call(*odd)
        assert torch.equal(want, got)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, plain, grad), torch.autograd.grad(got, odd, _odd_outer(grad))))


# ------------------------------------------------------------------------------------------------ gradients of gradients
def test_second_derivatives_are_refused():
    """create_graph=True gives the same first gradients; going through them again is an error, whether or not the incoming gradient itself asks
    for one."""
    dev = _dev()
    for name, call, x in _calls(dev, torch.float32):
        x = x.clone().requires_grad_()
        (want,) = torch.autograd.grad(call(x).square().sum(), x)
        (gx,) = torch.autograd.grad(call(x).square().sum(), x, create_graph=True)
        assert torch.equal(gx, want), name
        with pytest.raises(RuntimeError, match="second derivative"):
            gx.square().sum().backward()
        (gx,) = torch.autograd.grad(call(x).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            (gx.square().sum() + x.square().sum()).backward()
