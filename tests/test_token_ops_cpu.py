"""Token operators without a GPU: refusals of the Python and C entry points (all before any launch), and the oracle's own gradients."""
import math

import pytest
import torch

from oracle import ref_tokens as R


def test_python_refusals():
    from dose_prediction_amd import ops, _lib
    q = torch.zeros(2, 4, 6, 64)
    k = torch.zeros(2, 4, 3, 64)
    with pytest.raises(_lib.DoseHipError):
        ops.window_attention(q, k, k)                                   # no CPU fallback
    for bad in (dict(left=-1), dict(right=-2), dict(sinks=-1), dict(scale=0.0), dict(scale=math.nan), dict(q_start=1 << 31),
                dict(lengths=torch.tensor([4])), dict(lengths=torch.tensor([4.0, 4.0])), dict(q_start=torch.tensor([1, 2, 3]))):
        with pytest.raises(ValueError):
            ops.window_attention(q, k, k, **bad)
    for a, b, c in ((q, k[:, :, :, :32], k), (q, k, k[:, :3]), (q[:1], k, k), (q[0], k, k), (q, torch.zeros(2, 4, 4, 64), torch.zeros(2, 4, 4, 64)),
                    (q[..., :48], k[..., :48], k[..., :48])):
        with pytest.raises(ValueError):
            ops.window_attention(a, b, c)
    with pytest.raises(TypeError):
        ops.window_attention(q.double(), k.double(), k.double())
    x = torch.zeros(2, 4, 6 * 64)
    pos = torch.zeros(4, 3, dtype=torch.int32)
    for args, kw in (((x, 5, pos, (12, 10, 10)), {}), ((x, 12, pos, (12, 10, 11)), {}), ((x, 6, pos, (12, 10)), {}), ((x, 6, pos, (12, 10, 11)), {}),
                     ((x, 6, pos, (12, -1, 10)), {}), ((x, 6, pos[:3], (12, 10, 10)), {}), ((x, 6, pos, (12, 10, 10)), dict(base=1.0)),
                     ((x, 6, pos, None), {}), ((x[0], 6, pos, (12, 10, 10)), {}), ((x, 6, pos.expand(3, 4, 3), (12, 10, 10)), {})):
        with pytest.raises(ValueError):
            ops.rotary_axes(*args, **kw)
    with pytest.raises(TypeError):
        ops.rotary_axes(x, 6, pos.double(), (12, 10, 10))
    with pytest.raises(_lib.DoseHipError):
        ops.rotary_axes(x, 6, pos, (12, 10, 10))
    w = torch.ones(64)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(x, 3, 3, w, w, w, w.half())
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(x, 3, 3, w, w, w, w[:32])
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(x, 3, 3, w, w, w, w, sections=(12, 10, 10))
    with pytest.raises(ValueError):
        ops.window_attention_qkv(x, 2, 2, norm=(w, w))
    with pytest.raises(ValueError):
        ops.window_attention_qkv(x, 3, 2)
    with pytest.raises(_lib.DoseHipError):
        ops.window_attention_qkv(x, 2, 2, norm=(w, w, w, w), positions=pos, sections=(12, 10, 10))


def _fwd(**kw):
    a = dict(q=4096, k=4096, v=4096, o=4096, s=(0, 64, 64), B=1, heads=2, kv=1, Nq=4, Nk=4, d=64, left=1, right=1, sinks=0, scale=0.125, dtype=1, ws=0)
    a.update(kw)
    return ("dp_window_attention_fwd", a["q"], *a["s"], a["k"], *a["s"], a["v"], *a["s"], a["o"], *a["s"], 0, a["ws"], a["B"], a["heads"], a["kv"],
            a["Nq"], a["Nk"], a["d"], a["left"], a["right"], a["sinks"], 0, 0, 0, a["scale"], a["dtype"], 0)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dtype=-1), dict(d=80), dict(heads=3, kv=2), dict(kv=0), dict(Nq=-1), dict(Nk=-1), dict(B=-1),
                                 dict(left=-2), dict(right=-2), dict(sinks=-1), dict(scale=0.0), dict(scale=math.nan), dict(scale=-1.0),
                                 dict(q=4098), dict(v=4104), dict(s=(0, 60, 64)), dict(Nk=1 << 30), dict(Nq=1 << 29), dict(B=1 << 30),
                                 dict(Nq=1, Nk=1 << 20, left=-1)])
def test_c_refusals_of_window_attention(bad):
    """Answered before any launch (the last one: few queries over many keys need a workspace)."""
    from dose_prediction_amd import _lib
    with pytest.raises(_lib.DoseHipError):
        _lib.call(*_fwd(**bad))


def test_c_missing_pointers():
    from dose_prediction_amd import _lib
    for n in "qkvo":
        with pytest.raises(_lib.DoseHipError, match="missing"):
            _lib.call(*_fwd(**{n: 0}))
    mats = [(4096, 0, 64, 64)] * 5 + [(4096,), (4096,)] + [(4096, 0, 64, 64)] * 3
    for i in range(10):
        args = [m if j != i else (0, *m[1:]) for j, m in enumerate(mats)]
        with pytest.raises(_lib.DoseHipError, match="missing"):
            _lib.call("dp_window_attention_bwd", *(x for m in args for x in m), 0, 0, 1, 2, 1, 4, 4, 64, 1, 1, 0, 0, 0, 0, 0.125, 1, 0)
    for x, y in ((0, 4096), (4096, 0)):
        rot = (1, 4, 1, 1, 64)
        with pytest.raises(_lib.DoseHipError, match="missing"):
            _lib.call("dp_qk_rotary_fwd", x, 512, 128, y, 512, 128, *rot, 0, 0, 0, 0, 1e-5, 4096, 0, 0, 3, 12, 10, 10, 0, 10000.0, 0, 0, 1, 0)
        with pytest.raises(_lib.DoseHipError, match="missing"):
            _lib.call("dp_qk_rotary_bwd", 4096, 512, 128, x, 512, 128, 0, y, 512, 128, 0, 0, *rot, 0, 0, 1e-5, 4096, 0, 0, 3, 12, 10, 10, 0, 10000.0, 0,
                      1, 0)


def test_c_calls_without_work():
    from dose_prediction_amd import _lib
    assert _lib.call(*_fwd(B=0)) == 0 and _lib.call(*_fwd(Nq=0)) == 0
    mat = (4096, 0, 64, 64)
    assert _lib.call("dp_window_attention_bwd", *mat * 5, 4096, 4096, *mat * 3, 0, 0, 1, 2, 1, 0, 0, 64, 1, 1, 1, 0, 0, 0, 0.125, 1, 0) == 0
    L = _lib.lib()
    assert L.dp_window_attention_ws_elems(1, 2, 1, 0, 4, 64, 1, 1, 0, 0) == 0 and L.dp_window_attention_ws_elems(1, 2, 3, 4, 4, 64, 1, 1, 0, 1) == 0
    # a window without sinks never needs the sinks' partial sums, a long one with them does
    assert L.dp_window_attention_ws_elems(1, 12, 12, 8000, 8000, 64, 100, 100, 0, 1) == 0
    assert L.dp_window_attention_ws_elems(1, 12, 12, 8000, 8000, 64, 100, 100, 1, 1) > 0
    assert L.dp_window_attention_ws_elems(1, 12, 12, 8000, 8000, 64, -1, 100, 1, 1) == 0
    for t in (1, 7, 513, 100000, 1 << 33):
        assert 1 <= L.dp_qk_rotary_parts(t) <= 512


@pytest.mark.parametrize("bad", [dict(d=48), dict(dtype=5), dict(N=-1), dict(x=4100), dict(xt=100), dict(naxes=5), dict(naxes=0), dict(kind=3),
                                 dict(s0=33), dict(s1=21), dict(s0=-1), dict(base=1.0), dict(base=math.nan), dict(wq=4096), dict(wq=4096, bq=4100, wk=4096, bk=4096)])
def test_c_refusals_of_qk_rotary(bad):
    from dose_prediction_amd import _lib
    a = dict(x=4096, xt=128, N=4, d=64, wq=0, bq=0, wk=0, bk=0, kind=0, naxes=3, s0=12, s1=10, s2=10, base=10000.0, dtype=1)
    a.update(bad)
    with pytest.raises(_lib.DoseHipError):
        _lib.call("dp_qk_rotary_fwd", a["x"], 512, a["xt"], 4096, 512, 128, 1, a["N"], 1, 1, a["d"], a["wq"], a["bq"], a["wk"], a["bk"], 1e-5, 4096,
                  a["kind"], 0, a["naxes"], a["s0"], a["s1"], a["s2"], 0, a["base"], 0, 0, a["dtype"], 0)


def test_oracle_gradients_are_those_of_its_forward():
    """The formulas of ref_tokens.window's gradients against autograd through its own forward, in float64."""
    g = torch.Generator().manual_seed(3)
    q, k, v, go = (torch.randn(2, n, h, 32, generator=g, dtype=torch.float64) for n, h in ((11, 4), (9, 2), (9, 2), (11, 4)))
    kw = dict(left=3, right=2, sinks=1, start=torch.tensor([0, -2]), lengths=torch.tensor([9, 6]))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = R.window(*leaves, **kw)[0][0]
    auto = torch.autograd.grad(out, leaves, go)
    with torch.no_grad():
        form = R.window(*leaves, go, **kw)[1:]
    for a, (b, bound) in zip(auto, form):
        assert (a - b).abs().max().item() < 1e-12 and bool((bound >= 0).all())
    pos = torch.randint(0, 50, (7, 3), generator=g)
    x = torch.randn(1, 7, 2, 32, generator=g, dtype=torch.float64)
    for inter in (False, True):
        y = R.rotary(x, pos, (6, 5, 5), interleaved=inter)
        assert torch.allclose(R.rotary(y, -pos, (6, 5, 5), interleaved=inter), x, atol=1e-12) and torch.allclose(y.norm(dim=-1), x.norm(dim=-1))
