"""Token operators without a GPU: what reaches a call of them, with the launches replaced."""
import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    """The names of the entry points that a call launches; nothing is launched, any device's tensors pass."""
    from dose_prediction_amd import ops, _lib
    names = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: names.append(name) or 0)
    monkeypatch.setattr(ops, "_chk_dev", lambda *ts: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_device_of", lambda t: ops._NO_GUARD)
    return names


def _calls(N=9, heads=2, d=64):
    """(name, call of the packed projection)"""
    from dose_prediction_amd import ops
    pos = torch.zeros(N, 3, dtype=torch.int32)
    rot = dict(positions=pos, sections=(12, 10, 10))
    ws = [torch.ones(d) for _ in range(4)]

    def parts(t):
        return t.unflatten(-1, (3 * heads, d)).split(heads, 2)
    return [("rotary_axes", lambda t: ops.rotary_axes(t, 3 * heads, **rot)),
            ("qk_norm_rotary", lambda t: ops.qk_norm_rotary(t, heads, 2 * heads, *ws, **rot)),
            ("window_attention", lambda t: ops.window_attention(*parts(t), left=3)),
            ("window_attention_qkv", lambda t: ops.window_attention_qkv(t, heads, left=3, norm=ws, **rot))]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [False, True])
def test_recorded_calls_launch_when_they_are_replayed(launches, grad):
    for name, call in _calls():
        x = torch.zeros(2, 9, 6 * 64, requires_grad=grad)
        traced = torch.jit.trace(call, (x,), check_trace=False)
        del launches[:]
        call(x)
        want = list(launches)
        assert want
        for mode in (torch.no_grad, torch.enable_grad):
            del launches[:]
            with mode():
                traced(torch.ones_like(x))
            assert launches == want, name


@pytest.mark.filterwarnings("ignore")
def test_recorded_calls_check_the_sizes_of_the_replay(launches):
    """What the recording holds as constants (positions, lengths, weights) must fit the tensors that a replay brings, or nothing is launched."""
    from dose_prediction_amd import ops
    x, n = torch.zeros(2, 9, 6 * 64), torch.tensor([9, 3])
    pad = ("window_attention(lengths)", lambda t: ops.window_attention(*t.unflatten(-1, (6, 64)).split(2, 2), lengths=n))
    for name, call in [*_calls(), pad]:
        traced = torch.jit.trace(call, (x,), check_trace=False)
        del launches[:]
        for other in ((2, 12, 6 * 64), (2, 9, 6 * 32), (3, 9, 6 * 64)):
            if {"window_attention": True, pad[0]: other[0] == 2, "rotary_axes": other[1] == 9}.get(name, other == (3, 9, 6 * 64)):
                continue      # (these fit)
            with pytest.raises((ValueError, RuntimeError)):
                traced(torch.zeros(other))
            assert not launches, (name, other)


def test_forward_derivatives_are_refused(launches, monkeypatch):
    """Before any launch: a tangent is never dropped, whether or not torch says that a level of forward-mode derivatives is open."""
    from dose_prediction_amd import ops
    x = torch.zeros(2, 9, 6 * 64)
    for known in (True, False):
        if not known:
            monkeypatch.setattr(ops, "_fwd_ad", object())
        for name, call in _calls():
            with torch.autograd.forward_ad.dual_level():
                with pytest.raises(NotImplementedError, match="jvp"):
                    call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
            for transform in (lambda f: torch.func.jvp(f, (x,), (x,)), lambda f: torch.func.vjp(f, x)[1](x), lambda f: torch.func.vmap(f)(x.unsqueeze(0))):
                del launches[:]
                with pytest.raises(RuntimeError):
                    transform(call)
                assert not launches, name


@pytest.mark.parametrize("tiles", [False, True])
def test_strides_of_single_dimensions_are_not_handed_on(tiles):
    """Every stride that the kernels are given is a multiple of 16 bytes, or zero for a dimension of one; nothing is copied for it."""
    from dose_prediction_amd import ops
    base = torch.zeros(4096, dtype=torch.bfloat16)
    for shape, stride in (((1, 5, 2, 64), (999, 128, 64, 1)), ((1, 1, 2, 64), (999, 77, 64, 1)), ((2, 1, 1, 64), (64, 3, 5, 1)), ((1, 5, 64), (7, 64, 1)),
                          ((1, 1, 64), (7, 9, 1)), ((2, 5, 64), (320, 64, 1))):
        t = base.as_strided(shape, stride)
        assert t.is_contiguous()
        same, st = ops._strided(t, tiles)
        assert same is t and list(st) == [0 if n == 1 else s for n, s in zip(shape[:-1], stride)], shape
        odd = torch.zeros(4097, dtype=torch.bfloat16)[1:].as_strided(shape, stride)      # (a row that is not aligned: copied)
        copy, st = ops._strided(odd, tiles)
        assert copy.data_ptr() % 16 == 0 and copy.shape == odd.shape and all(n == 1 or x % 8 == 0 for n, x in zip(shape, st)), shape
        assert all(x % 8 == 0 for x in st), (shape, st)


def test_second_derivatives_are_refused_where_the_incoming_gradient_has_no_graph(launches):
    """The gradient of a sum's argument is constant, that of its inputs is not: the refusal hangs on none of them."""
    for name, call in _calls():
        for loss in (lambda y: y.sum(), lambda y: y.square().sum()):
            x = torch.zeros(2, 9, 6 * 64, requires_grad=True)
            (gx,) = torch.autograd.grad(loss(call(x)), x, create_graph=True)
            with pytest.raises(RuntimeError, match="second derivative"):
                (gx.sum() + x.square().sum()).backward()
            (gx,) = torch.autograd.grad(loss(call(x)), x)
            assert not gx.requires_grad


def test_a_norm_with_a_part_missing_is_refused():
    from dose_prediction_amd import ops
    x, w = torch.zeros(2, 9, 6 * 64), torch.ones(64)
    for i in range(4):
        for have in ([w] * 4, [None] * 4):
            part = list(have)
            part[i] = None if have[0] is w else w
            with pytest.raises(ValueError, match="None"):
                ops.window_attention_qkv(x, 2, norm=part)
            with pytest.raises(ValueError, match="None"):
                ops.qk_norm_rotary(x, 2, 4, *part)


def test_weights_on_another_device_are_refused(launches):
    """(The kernels would read them through an address of the other device.)"""
    from dose_prediction_amd import ops, _lib
    x = torch.zeros(2, 9, 6 * 64)
    for i in range(4):
        ws = [torch.ones(64, device="meta" if j == i else "cpu") for j in range(4)]
        for grad in (False, True):
            y = x.clone().requires_grad_(grad)
            with pytest.raises(_lib.DoseHipError, match="on meta"):
                ops.window_attention_qkv(y, 2, norm=ws)
            with pytest.raises(_lib.DoseHipError, match="on meta"):
                ops.qk_norm_rotary(y, 2, 4, *ws)
    assert not launches


def test_networks_pickled_before_the_options_run_as_they_did(monkeypatch):
    """A whole network that was stored without the attention's options comes back with full attention."""
    import pickle
    from dose_prediction_amd import blocks, ops
    calls = []
    for name, out in (("linear", lambda x, *a, **k: x), ("layer_norm", lambda x, *a: x), ("add_layer_norm", lambda x, y, *a: (x, y)), ("add", lambda x, y: x),
                      ("attention", lambda x, heads: calls.append(heads) or x), ("gelu", lambda x: x), ("mlp", lambda x, *a, **k: x)):
        if hasattr(ops, name):
            monkeypatch.setattr(ops, name, out)
    monkeypatch.setattr(blocks.PatchEmbeddingBlock, "forward", lambda self, x: x)
    monkeypatch.setattr(blocks.MLPBlock, "forward", lambda self, x: x)
    net = blocks.ViT(1, (32, 32, 32), (16, 16, 16), hidden_size=64, mlp_dim=64, num_layers=2, num_heads=2, pos_embed="perceptron")
    del net._buffers["positions"]
    net._non_persistent_buffers_set.discard("positions")
    for blk in net.blocks:
        for name in ("full", "rotary", "left", "right", "sinks", "qk_norm", "base", "interleaved"):
            del blk.attn.__dict__[name]
    old = pickle.loads(pickle.dumps(net))
    x = torch.zeros(1, 8, 64)
    n, hidden = old(x)
    assert n is x and len(hidden) == 2 and calls == [2, 2]
    assert old.blocks[0](x) is x and calls == [2, 2, 2]
