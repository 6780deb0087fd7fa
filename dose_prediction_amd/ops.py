"""torch.autograd.Function wrappers over the C ABI (include/dose_hip.h).

Tensor conventions inside the HIP path
  * activations: 5-D ``[N, D, H, W, C]`` (NDHWC), last stride 1; a tensor may be a channel slice of a
    wider buffer (row pitch ``ld`` = stride of W).  dtype float32 (parity mode), bfloat16 (bench mode) or float16.
  * token matrices: 2-D/3-D ``[..., rows, C]`` contiguous.
  * parameters stay fp32 ``nn.Parameter``s in the reference's own shapes (state_dict compatible); kernels
    consume packed copies cached per (parameter version, dtype).  Weight gradients are produced in fp32.
PyTorch only provides device memory, the current stream and autograd bookkeeping here.
"""
import functools
import math
import os

import torch
from torch.autograd import forward_ad as _fwd_ad

from . import _lib

ACT = {None: 0, "none": 0, "relu": 1, "lrelu": 2, "mish": 3, "gelu": 4}
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _act_code(act, dtype=None):
    """Activation code of the normalisation kernels; Mish on fp32 tensors in the fp32x3 mode uses the hardware exp2 / rcp forms
    (DP_ACT_MISH_FAST: ~1e-7 relative, as the 16-bit modes always do)."""
    if act == "mish" and dtype == torch.float32:
        from . import config
        if config.x3():
            return 5
    return ACT[act]


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream():
    """The current HIP stream as an integer handle (the launch thread has to stay ahead of the GPU: torch.cuda.current_stream() builds
    a Stream object through three Python layers, 8 us x 750 launches per step)."""
    if _raw_stream is not None:
        return _raw_stream(_raw_device())
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return 0 if t is None else t.data_ptr()


def _dt(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"HIP path supports float32/bfloat16/float16 activations, got {t.dtype}")


def _chk_dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise _lib.DoseHipError("dose_prediction_amd ops need CUDA/HIP tensors (there is no CPU fallback)")


def rows_ld(t):
    """(rows, C, ld) of an activation / matrix whose rows are uniformly pitched."""
    if t.is_contiguous() and t.dim() > 0:    # (the common case in ~0.3 us: this runs ~720 times per training step, tools/host_profile.py)
        C = t.shape[-1]
        return (t.numel() // C if C else 0), C, C
    shape, st = t.shape, t.stride()
    C, nd = shape[-1], len(shape)
    if st[-1] != 1 and C > 1:
        raise ValueError("last dim must be contiguous")
    if nd == 1:
        return 1, C, C
    ld = st[-2] if shape[-2] > 1 else max(C, st[-2])
    rows = 1
    exp = ld
    for d in range(nd - 2, -1, -1):
        n = shape[d]
        if n > 1 and st[d] != exp:
            raise ValueError(f"tensor is not a uniformly pitched row matrix: shape {tuple(shape)} strides {st}")
        exp *= n
        rows *= n
    return rows, C, ld


def as_rows(t):
    """Return a tensor satisfying rows_ld (copying if needed)."""
    try:
        rows_ld(t)
        return t
    except ValueError:
        return t.contiguous()


def new_act(like, shape, dtype=None):
    return torch.empty(shape, dtype=dtype or like.dtype, device=like.device)


# ------------------------------------------------------------------------------------------------ packed-weight cache
class _PackCache:
    """Packed (kernel-layout) copies of a parameter, stored ON the parameter object so that their lifetime is the
    parameter's; an entry is rebuilt when the parameter's version counter, storage, device or pack generation changed
    (optimizer.step(), load_state_dict(), .to()).  Updates that bypass autograd's version counter (FusedAdam writes through raw
    pointers, the DDP broadcast through .data) MUST call refresh_packs() / invalidate_packs() on the parameters they touched.

    Entry: [tag, packed tensor, descriptor, used-since-last-refresh].  The descriptor (kind, a, b, c, d, e) is the dp_pack_multi
    table row that rebuilds the copy in place; None = the copy aliases the parameter or can only be rebuilt by its builder."""

    @staticmethod
    def tag(w):
        return (w._version, w.data_ptr(), w.device, w.__dict__.get("_dp_gen", 0))

    def get(self, w, key, builder, desc=None):
        store = w.__dict__.setdefault("_dp_packs", {})
        ent = store.get(key)
        tag = self.tag(w)
        if ent is None or ent[0] != tag:
            dst = builder()
            ent = [tag, dst, desc(dst) if (desc is not None and w.is_contiguous()) else None, True]
            store[key] = ent
        ent[3] = True
        return ent[1]


_packs = _PackCache()
_REPACK_PLANS = {}


def unscale_grads(params):
    """Divide the gradients of ``params`` by config.effective_loss_scale() in one multi-tensor pass (for optimizers other than FusedAdam,
    which unscales inside its kernel)."""
    from . import config
    gs = [p.grad for p in params if p.grad is not None]
    if gs and config.effective_loss_scale() != 1.0:
        torch._foreach_mul_(gs, 1.0 / config.effective_loss_scale())


def invalidate_packs(params):
    """Drop every packed copy of ``params`` (they are rebuilt lazily by the next forward)."""
    for p in params:
        p.__dict__.pop("_dp_packs", None)
        p.__dict__["_dp_gen"] = p.__dict__.get("_dp_gen", 0) + 1


def adam_fusable_pack(p):
    """(key, dst pointer, ckind, K, cpp) of ONE packed copy of ``p`` that dp_adam_multi can write itself while it updates p (the
    layouts that follow the parameter's own element order: plain 16-bit casts and fp32x3 Linear operands), or (None, 0, 0, 0, 0)."""
    store = p.__dict__.get("_dp_packs")
    if store and p.is_contiguous() and p.numel() < (1 << 32):
        for key, ent in store.items():
            dst, d = ent[1], ent[2]
            if d is None or not ent[3] or dst.data_ptr() == p.data_ptr() or ent[0][1:3] != (p.data_ptr(), p.device):
                continue
            base, pat, cp = d[0] & 0xff, (d[0] >> 8) & 0xff, d[0] >> 16
            if base == 0 and cp == 0 and dst.dtype in (torch.bfloat16, torch.float16) and dst.numel() == p.numel():
                return key, dst.data_ptr(), 1 if dst.dtype == torch.bfloat16 else 2, 0, 0
            if base == 1 and cp > 0 and d[3] == 3 * cp and d[2] % 4 == 0 and d[1] * d[2] == p.numel() and dst.dtype == torch.bfloat16:
                return key, dst.data_ptr(), 3, d[2], cp | (pat << 32)
    return None, 0, 0, 0, 0


def _pack_chunks(L, desc, dst, chunk):
    """Blocks dp_pack_multi needs for one table row (dp_pack_chunks; fp32 destinations keep the element walk)."""
    if dst.element_size() == 2 or (desc[0] & 0xff) == 2:
        return int(L.dp_pack_chunks(desc[0], desc[1], desc[2], desc[3], desc[4], desc[5], dst.numel()))
    return -(-dst.numel() // chunk)


def refresh_packs(params, fused=None):
    """Rebuild, in ONE launch per storage type (dp_pack_multi), every packed copy of ``params`` that was used since the last
    refresh; called by FusedAdam.step() right after the update kernel, which changes the parameters through raw pointers
    (p._version does not move).  Copies that were not used since the last refresh are dropped.  fused: {id(p): key} of the copies
    the update kernel has already rewritten itself (adam_fusable_pack)."""
    L = _lib.lib()
    chunk = L.dp_pack_chunk()
    jobs = {}
    for p in params:
        store = p.__dict__.get("_dp_packs")
        p.__dict__["_dp_gen"] = p.__dict__.get("_dp_gen", 0) + 1
        if not store:
            continue
        tag = _packs.tag(p)
        for key in list(store):
            ent = store[key]
            dst = ent[1]
            if dst.data_ptr() == p.data_ptr():          # the "copy" is the parameter itself (fp32 row-major matrix)
                ent[0] = tag
                continue
            if fused and fused.get(id(p)) == key:       # written by dp_adam_multi together with the parameter
                ent[0], ent[3] = tag, False
                continue
            if ent[2] is None or not ent[3] or ent[0][1:3] != tag[1:3]:
                del store[key]
                continue
            ent[0], ent[3] = tag, False
            jobs.setdefault((dst.dtype, dst.device), []).append((p, dst, ent[2]))
    for (dtype, dev), lst in jobs.items():
        pkey = (dtype, dev, tuple((p.data_ptr(), d.data_ptr()) for p, d, _ in lst))
        plan = _REPACK_PLANS.get(pkey)
        if plan is None:
            rows, ct, ci = [], [], []
            for t, (p, d, desc) in enumerate(lst):
                kind, a, b, c = desc[0], desc[1], desc[2], desc[3]
                rows.append((p.data_ptr(), d.data_ptr()) + tuple(desc))
                n = _pack_chunks(L, desc, d, chunk)
                ct += [t] * n
                ci += list(range(n))
            plan = (torch.tensor(rows, dtype=torch.int64, device=dev), torch.tensor(ct, dtype=torch.int32, device=dev),
                    torch.tensor(ci, dtype=torch.int32, device=dev), len(ct))
            if len(_REPACK_PLANS) > 16:
                _REPACK_PLANS.clear()
            _REPACK_PLANS[pkey] = plan
        _lib.call("dp_pack_multi", _p(plan[0]), _p(plan[1]), _p(plan[2]), plan[3], _DT[dtype], _stream())


def _pack_conv(w, mode, dtype):
    """torch [Cout,Cin,k,k,k] fp32 -> packed T (see dp_pack_conv_weight)."""
    cout, cin = w.shape[0], w.shape[1]
    taps = w[0, 0].numel()

    def build():
        rows, inner = (cout, cin) if mode == 0 else (cin, cout)
        dst = torch.empty((rows, taps, (inner + 7) // 8 * 8), dtype=dtype, device=w.device)
        wc = w.detach().contiguous()
        _lib.call("dp_pack_conv_weight", _p(wc), _p(dst), cout, cin, taps, mode, _DT[dtype], _stream())
        return dst
    return _packs.get(w, ("conv", mode, dtype), build, lambda dst: (3, cout, cin, taps, mode, 0))


USE_TILED = True


def _tiled_elems(cin, cout, k, stride, pad, dil, W):
    if not USE_TILED:
        return 0
    return _lib.lib().dp_conv3d_tiled_weight_elems(cin, cout, k, stride, pad, dil, W)


_ZERO_SCRATCH = {}


def _zero_scratch(device, n):
    """Persistent all-zero fp32 scratch for the kernels that accumulate with atomics (dp_scratch_contract(1): they get it zeroed and
    hand it back zeroed, so no memset launch per call).  One buffer per (device, stream), grown on demand: two streams issuing
    atomically-accumulating kernels concurrently never share a scratch."""
    L = _lib.lib()
    key = (device.type, device.index, _stream())
    buf = _ZERO_SCRATCH.get(key)
    if buf is None or buf.numel() < n:
        buf = torch.zeros((max(n, 1 << 22),), dtype=torch.float32, device=device)
        _ZERO_SCRATCH[key] = buf
        L.dp_scratch_contract(1)
    return buf


# Weight-gradient destinations registered by the data-parallel reducer (dose_prediction_amd.ddp): parameter data_ptr -> callable
# returning a fresh fp32 view of the parameter's slot in its flat all-reduce bucket (or None).  The weight-gradient kernels then
# write straight into the bucket and autograd adopts the view as .grad, so no pack copy is needed before the exchange.
GRAD_DEST = {}


_ZERO_POOL = {}


def _zero_bias_grad(bias):
    """An all-zero fp32 gradient for a bias whose gradient is identically zero (bias_grad_zero): a persistent per-parameter slice of
    one zero buffer per device instead of a fill launch per layer and step.  Optimizers only read gradients and zero_grad / scaling /
    accumulating another such gradient leave zeros zero; the pool is wiped once per backward pass in case somebody did write."""
    dev = bias.device
    pool = _ZERO_POOL.get(dev)
    if pool is None:
        pool = _ZERO_POOL[dev] = {"buf": torch.zeros((1 << 16,), dtype=torch.float32, device=dev), "used": 0, "slots": {}}
    key = (bias.data_ptr(), bias.numel())
    off = pool["slots"].get(key)
    n = bias.numel()
    if off is None:
        if pool["used"] + n > pool["buf"].numel():
            return torch.zeros(bias.shape, dtype=torch.float32, device=dev)
        off = pool["slots"][key] = pool["used"]
        pool["used"] += (n + 63) // 64 * 64
    task = _graph_task_id()
    if not pool.get("armed") or _pass_is_stale(pool, task):
        # first hand-out of this backward pass: wipe the pool (one 256 KB fill), so that whatever was written into a previous step's
        # .grad in place (a regulariser's grad.add_, a NaN from clip_grad_norm_) cannot survive into this step; a pass
        # that raised before its end-of-backward callback leaves "armed" behind -- _pass_is_stale tells
        pool["buf"].zero_()
        pool["armed"], pool["task"], pool["epoch"] = True, task, _FWD_EPOCH[0]
        torch.autograd.Variable._execution_engine.queue_callback(lambda: pool.__setitem__("armed", False))
    # a FRESH view object every time: autograd adopts it as .grad without a copy only if nobody else holds the tensor object
    return pool["buf"][off:off + n].view(bias.shape)


_PASS_ARENA = {}
_PASS_ARENA_ON = os.environ.get("DOSE_HIP_PASS_ARENA", "1") != "0"      # (A/B switch)
_PASS_ARENA_MAX_ELEMS = 1 << 20
_graph_task_id = getattr(torch._C, "_current_graph_task_id", lambda: -1)      # id of the running backward pass (-1 outside one)
_FWD_EPOCH = [0]        # bumped by the network-entry conversion (ToNDHWC.forward) whenever it runs OUTSIDE any backward pass


def _pass_is_stale(state, task):
    """state was armed by backward pass state["task"] and never disarmed; the request comes from pass `task`.  A different id alone does
    not make the armed pass dead: a NESTED backward (reentrant activation checkpointing, torch.autograd.grad inside a backward node) has
    an id of its own while the outer pass is suspended, and resetting there re-allocates / re-fills once per segment.  The
    armed pass is known to be dead when a network forward has started outside every backward pass since it armed (its end-of-backward
    callback would have run first had it ended normally)."""
    return state.get("task") != task and state.get("epoch") != _FWD_EPOCH[0]


def _pass_zeros(shape, dev):
    """A zero-filled fp32 tensor for an accumulator of the backward pass (LayerNorm's dgamma / dbeta, split-K weight gradients):
    a slice of ONE arena per device and backward pass, filled by one launch at its first use (the pass used to issue ~30 five-microsecond
    fill launches, each waiting its turn behind full-chip kernels on the critical stream).  The arena is a FRESH
    tensor every pass -- gradients handed to autograd as views of it keep it alive, so accumulation over several backward passes is
    safe -- sized by what the previous pass asked for; requests beyond it get their own torch.zeros.  Only call from backward functions."""
    n = 1
    for d in shape:
        n *= int(d)
    if dev.type != "cuda" or n == 0 or not _PASS_ARENA_ON:
        return torch.zeros(shape, dtype=torch.float32, device=dev)
    if n > _PASS_ARENA_MAX_ELEMS:
        # (a gradient adopted as a view of the arena pins the WHOLE arena until every such gradient is released: big accumulators --
        # split-K dW buffers of tens of MB -- get their own allocation)
        return torch.zeros(shape, dtype=torch.float32, device=dev)
    a = _PASS_ARENA.get(dev)
    if a is None:
        a = _PASS_ARENA[dev] = {"buf": None, "used": 0, "need": 0, "now": 0, "armed": False, "ev": None, "stream": None, "task": None}
    task = _graph_task_id()
    if a["armed"] and _pass_is_stale(a, task):
        # the pass that armed the arena never reached its end-of-backward callback (it raised): start over.  A nested pass
        # keeps drawing from the outer pass's arena: slices that were never handed out are still zero whoever asks.
        a["armed"], a["buf"] = False, None
    if not a["armed"]:
        a["buf"] = torch.zeros((max(a["need"], 1 << 16),), dtype=torch.float32, device=dev)
        a["used"], a["now"], a["armed"], a["task"], a["epoch"] = 0, 0, True, task, _FWD_EPOCH[0]
        a["stream"] = _current_stream_object(dev)
        a["ev"] = torch.cuda.Event()
        a["ev"].record(a["stream"])

        def _end(a=a):
            a["armed"], a["need"], a["buf"] = False, max(a["need"], a["now"]), None
        torch.autograd.Variable._execution_engine.queue_callback(_end)
    step = (n + 63) // 64 * 64
    a["now"] += step
    if a["used"] + step > a["buf"].numel():
        return torch.zeros(shape, dtype=torch.float32, device=dev)
    t = a["buf"][a["used"]:a["used"] + n].view(shape)
    a["used"] += step
    cur = _current_stream_object(dev)
    if cur != a["stream"]:
        cur.wait_event(a["ev"])           # (the fill ran on the stream of the pass's first request)
        a["buf"].record_stream(cur)
    return t


def _wgrad_buffer(weight, zero):
    f = GRAD_DEST.get(weight.data_ptr()) if GRAD_DEST else None
    buf = f() if f is not None else None
    if buf is None:
        return _pass_zeros(weight.shape, weight.device) if zero else torch.empty(weight.shape, dtype=torch.float32, device=weight.device)
    return buf.zero_() if zero else buf


def _tiled_ws(like, N, D, H, W, cin, cout, k):
    n = _lib.lib().dp_conv3d_tiled_ws_elems(N, D, H, W, cin, cout, k)
    if n < 0:
        raise _lib.DoseHipError("conv3d_tiled: scratch too large")
    return _zero_scratch(like.device, n) if n else None


def _pack_conv_tiled(w, tf, dtype, elems, W):
    """Weights for the LDS-tiled conv kernels (tf=1: transposed+flipped, i.e. the data-gradient convolution); W = row length of
    the volume the convolution runs on (selects the 32x32x16 or the 16x16x32 kernel's layout: dp_conv3d_tiled_layout)."""
    k = w.shape[2]
    co, ci = (w.shape[1], w.shape[0]) if tf else (w.shape[0], w.shape[1])      # roles in the convolution being computed
    layout = _lib.lib().dp_conv3d_tiled_layout(ci, co, k, 1, k // 2, 1, W)
    fn = "dp_pack_conv_weight_cc16" if layout == 2 else "dp_pack_conv_weight_tiled"

    def build():
        dst = torch.empty((elems,), dtype=dtype, device=w.device)
        wc = w.detach().contiguous()
        _lib.call(fn, _p(wc), _p(dst), co, ci, k, 1 if tf else 0, _DT[dtype], _stream())
        return dst

    def desc(dst):
        if layout == 2:
            return (6, co, ci, k, 0, 1 if tf else 0)
        return (4, co, ci, k, _lib.lib().dp_conv3d_tiled_npair(co), 1 if tf else 0)
    return _packs.get(w, ("conv_tiled", tf, dtype, elems, layout), build, desc)


def _pack_tconv(w, transposed, dtype):
    """ConvTranspose3d weight [Cin,Cout,2,2,2] -> [(abc,co)][CinP] (fwd) or [Cin][(abc,co)P] (data grad)."""
    def build():
        cin, cout = w.shape[0], w.shape[1]
        m = w.detach().permute(2, 3, 4, 1, 0).reshape(8 * cout, cin)      # [(abc,co), ci]
        if transposed:
            m = m.t()
        m = m.contiguous()
        pad = (-m.shape[1]) % 8
        dst = torch.zeros((m.shape[0], m.shape[1] + pad), dtype=dtype, device=w.device)
        tmp = torch.empty(m.shape, dtype=dtype, device=w.device)
        _lib.call("dp_cast", _p(m), 0, _p(tmp), _DT[dtype], m.numel(), _stream())
        _lib.call("dp_copy_rows", _p(tmp), m.shape[1], _p(dst), dst.shape[1], m.shape[0], m.shape[1], _DT[dtype], _stream())
        return dst
    return _packs.get(w, ("tconv", transposed, dtype), build,
                      lambda dst: (5, w.shape[0], w.shape[1], dst.shape[1], 1 if transposed else 0, 0))


def _pack_mat(w, transposed, dtype):
    """Linear weight [out,in] fp32 -> T [out][inP] or (transposed) [in][outP]."""
    def build():
        m = w.detach()
        m = (m.t() if transposed else m).contiguous()
        pad = (-m.shape[1]) % 8
        if pad == 0 and dtype == torch.float32:
            return m
        dst = torch.zeros((m.shape[0], m.shape[1] + pad), dtype=dtype, device=w.device)
        tmp = torch.empty(m.shape, dtype=dtype, device=w.device)
        _lib.call("dp_cast", _p(m), 0, _p(tmp), _DT[dtype], m.numel(), _stream())
        _lib.call("dp_copy_rows", _p(tmp), m.shape[1], _p(dst), dst.shape[1], m.shape[0], m.shape[1], _DT[dtype], _stream())
        return dst
    def desc(dst):
        if transposed:
            return (2, w.shape[1], w.shape[0], dst.shape[1], 0, 0)
        if dst.shape[1] == w.shape[1]:
            return (0, w.numel(), 0, 0, 0, 0)
        return (1, w.shape[0], w.shape[1], dst.shape[1], 0, 0)
    return _packs.get(w, ("mat", transposed, dtype), build, desc)


def _cast_vec(v, dtype):
    if v is None or v.dtype == dtype:
        return v
    out = torch.empty(v.shape, dtype=dtype, device=v.device)
    vc = v.detach().contiguous()
    _lib.call("dp_cast", _p(vc), _DT[vc.dtype], _p(out), _DT[dtype], vc.numel(), _stream())
    return out


# ------------------------------------------------------------------------------------------------ raw helpers
_PW_MAXK = int(os.environ.get("DOSE_HIP_PW_MAXK", "64"))


def gemm_nt(A, B, out, bias=None, alpha=1.0, M=None, N=None, K=None, batch=(1, 1), sa=(0, 0), sb=(0, 0), sc=(0, 0),
            lda=None, ldb=None, ldc=None, splitk=1, x3_terms=None):
    """out[m][n] = alpha * sum_k A[m][k] B[n][k] (+bias).  A, B share dtype; out dtype float32 => fp32 output.
    x3_terms (fp32 operands in the fp32x3 mode only): 3 / 1 = the caller accepts split-bf16 products (three: forward passes, one: the
    one-product data gradients) where the matrix-core row kernel takes the shape; None = exact fp32 arithmetic."""
    out_f32 = 1 if (out.dtype == torch.float32 and A.dtype != torch.float32) or splitk > 1 else 0
    if splitk > 1 and out.dtype != torch.float32:
        raise ValueError("split-K needs an fp32 output")
    if batch == (1, 1) and splitk == 1 and not out_f32 and alpha == 1.0 and M >= 32768 and out.dtype == A.dtype:
        # millions of voxel rows x a handful of channels: a row stream, not a tiled GEMM -- the matrix-core row kernel where it applies
        # (16-bit storage, up to 256 input channels: pointwise convolutions, ConvTranspose data gradients), the VALU stream otherwise
        if ((K <= _PW_MAXK and N <= 32) or (A.dtype != torch.float32 and K <= 256 and _p(A) % 16 == 0 and _p(out) % 16 == 0
                                            and _lib.lib().dp_rows_mfma_ok(lda, ldb, ldc, K, N, _dt(A)))):
            _lib.call("dp_pointwise_rows", _p(A), lda, _p(B), ldb, _p(bias), _p(out), ldc, M, K, N, _dt(A), _stream())
            return
        xdt = {3: DP_X3, 1: DP_X1}.get(x3_terms)
        if (xdt is not None and A.dtype == torch.float32 and K <= 128 and _p(A) % 16 == 0 and _p(out) % 16 == 0
                and _lib.lib().dp_rows_mfma_ok(lda, ldb, ldc, K, N, xdt)):
            # fp32x3: fp32 rows split into bf16 halves in registers (k_rows_mfma_f32) instead of the exact-fp32 tiled GEMM
            _lib.call("dp_pointwise_rows", _p(A), lda, _p(B), ldb, _p(bias), _p(out), ldc, M, K, N, xdt, _stream())
            return
    _lib.call("dp_gemm_nt", _p(A), lda, sa[0], sa[1], _p(B), ldb, sb[0], sb[1], _p(out), ldc, sc[0], sc[1], _p(bias),
              M, N, K, batch[0], batch[1], float(alpha), out_f32, splitk, _dt(A), _stream())


def _gemm_nt_splitk_det(A, B, bias, rows, nout, K, lda, ldb, splitk):
    """Deterministic split-K (config.set_deterministic): the K shares as a BATCHED GEMM into their own [rows, nout] fp32 slabs, added in
    order (torch.sum over the leading axis is order-fixed) -- instead of fp32 atomics into one matrix, and without giving up the
    parallelism over K (unsplit, the patch embedding's K = 102 400 runs on 48 tiles).  Returns the fp32 [rows, nout] result or None when
    the shares cannot be cut on 16-byte boundaries (the caller then lets the library run it unsplit)."""
    ks = K // splitk
    if splitk < 2 or ks * splitk != K or ks % 8 or lda != K or ldb < K:
        return None
    parts = torch.empty((splitk, rows, nout), dtype=torch.float32, device=A.device)
    gemm_nt(A, B, parts, M=rows, N=nout, K=ks, batch=(splitk, 1), sa=(ks, 0), sb=(ks, 0), sc=(rows * nout, 0), lda=lda, ldb=ldb, ldc=nout)
    acc = parts.sum(0)
    return acc if bias is None else acc.add_(bias)


def _x3_terms(forward):
    """Split products a contraction may use in the CURRENT mode: None outside fp32x3 (exact arithmetic of the storage type), 3 for a
    forward pass, config.x3_dgrad_terms() for a data gradient."""
    from . import config
    if not config.x3():
        return None
    return 3 if forward else config.x3_dgrad_terms()


def colsum_into(gy2d_rows, ld, rows, C, db, dtype_code):
    """db[c] = sum_rows gy[row][c]  (stats partial + batch-mode finalize, which overwrites: db need not be initialised)."""
    L = _lib.lib()
    nblk = L.dp_stats_nblk(rows)
    es = 4 if dtype_code == 0 else 2
    step = 2048                               # the row-stream kernels handle up to 2048 channels per launch
    for c0 in range(0, C, step):
        c = min(step, C - c0)
        part = torch.empty((nblk, 2, c), dtype=torch.float32, device=db.device)
        s = torch.empty((2, c), dtype=torch.float32, device=db.device)
        _lib.call("dp_stats_partial", gy2d_rows + c0 * es, ld, 1, rows, c, _p(part), dtype_code, _stream())
        _lib.call("dp_norm_bwd_finalize", _p(part), 1, nblk, c, 1, _p(s[0]), _p(s[1]), 0, db.data_ptr() + 4 * c0, _stream())


def wgrad(x, ldx, gy, ldgy, dw, geom, cin, cout, k, stride, pad, dil, shift, choff, s_co, s_ci, s_tap, dtype_code):
    N, Di, Hi, Wi, Do, Ho, Wo = geom
    _lib.call("dp_conv3d_wgrad", _p(x), ldx, _p(gy), ldgy, _p(dw), N, Di, Hi, Wi, Do, Ho, Wo, cin, cout, k, stride, pad, dil,
              shift, choff, s_co, s_ci, s_tap, dtype_code, _stream())


# ------------------------------------------------------------------------------------------------ layout
class ToNDHWC(torch.autograd.Function):
    """NCDHW fp32 (the trainer's tensors, network_trainer.py:230) -> NDHWC T, channels zero-padded to cpad."""

    @staticmethod
    def forward(ctx, x, cpad, dtype):
        _chk_dev(x)
        if _graph_task_id() == -1:
            _FWD_EPOCH[0] += 1          # a network forward outside any backward pass: whatever pass state is still armed is dead (_pass_is_stale)
        x = x.contiguous().float()
        N, C = x.shape[:2]
        sp = tuple(x.shape[2:])
        V = sp[0] * sp[1] * sp[2]
        y = torch.empty((N,) + sp + (cpad,), dtype=dtype, device=x.device)
        _lib.call("dp_ncdhw_to_ndhwc", _p(x), _p(y), N, C, V, cpad, cpad, _DT[dtype], _stream())
        ctx.C = C
        return y

    @staticmethod
    def backward(ctx, gy):
        gy = as_rows(gy)
        rows, cp, ld = rows_ld(gy)
        N = gy.shape[0]
        sp = tuple(gy.shape[1:4])
        gx = torch.empty((N, ctx.C) + sp, dtype=torch.float32, device=gy.device)
        _lib.call("dp_ndhwc_to_ncdhw", _p(gy), _p(gx), N, ctx.C, rows // N, ld, 0, _dt(gy), _stream())
        from . import config
        if config.effective_loss_scale() != 1.0 and gy.dtype != torch.float32:
            gx = gx / config.effective_loss_scale()
        return gx, None, None


class FromNDHWC(torch.autograd.Function):
    """NDHWC T -> NCDHW fp32 (what the loss / trainer consume)."""

    @staticmethod
    def forward(ctx, x):
        _chk_dev(x)
        x = as_rows(x)
        rows, C, ld = rows_ld(x)
        N = x.shape[0]
        sp = tuple(x.shape[1:4])
        y = torch.empty((N, C) + sp, dtype=torch.float32, device=x.device)
        _lib.call("dp_ndhwc_to_ncdhw", _p(x), _p(y), N, C, rows // N, ld, 0, _dt(x), _stream())
        ctx.dtype = x.dtype
        return y

    @staticmethod
    def backward(ctx, gy):
        gy = gy.contiguous().float()
        from . import config
        if config.effective_loss_scale() != 1.0 and ctx.dtype != torch.float32:
            gy = gy * config.effective_loss_scale()         # loss scaling enters the 16-bit domain here (config.set_loss_scale)
        N, C = gy.shape[:2]
        sp = tuple(gy.shape[2:])
        gx = torch.empty((N,) + sp + (C,), dtype=ctx.dtype, device=gy.device)
        _lib.call("dp_ncdhw_to_ndhwc", _p(gy), _p(gx), N, C, sp[0] * sp[1] * sp[2], C, C, _DT[ctx.dtype], _stream())
        return gx


class Cat(torch.autograd.Function):
    """torch.cat(dim=channels) by strided row copies; backward hands out channel-slice views."""

    @staticmethod
    def forward(ctx, *xs):
        xs = [as_rows(x) for x in xs]
        cs = [x.shape[-1] for x in xs]
        out = torch.empty(tuple(xs[0].shape[:-1]) + (sum(cs),), dtype=xs[0].dtype, device=xs[0].device)
        if len(xs) == 2 and cs[0] % 8 == 0:
            (rows, _, lda), (_, _, ldb) = rows_ld(xs[0]), rows_ld(xs[1])
            _lib.call("dp_cat2_rows", _p(xs[0]), lda, cs[0], _p(xs[1]), ldb, cs[1], _p(out), out.shape[-1], rows, _dt(out), _stream())
        else:
            off = 0
            for x, c in zip(xs, cs):
                rows, _, ld = rows_ld(x)
                _lib.call("dp_copy_rows", _p(x), ld, out.data_ptr() + off * out.element_size(), out.shape[-1], rows, c, _dt(x), _stream())
                off += c
        ctx.cs = cs
        return out

    @staticmethod
    def backward(ctx, g):
        outs, off = [], 0
        for c in ctx.cs:
            outs.append(g[..., off:off + c])
            off += c
        return tuple(outs)


def cat(xs):
    return Cat.apply(*xs)


# ------------------------------------------------------------------------------------------------ weight-gradient stream
_WG = {"dirty": {}, "queued": False}


_STREAM_OBJ = {}


def _current_stream_object(dev=None):
    """torch.cuda.current_stream(dev), cached by raw handle: the stock call goes through three Python layers (device-index resolution,
    is_available, the Stream constructor: ~9 us), and the reducer's per-parameter hooks alone made it 220 times per step (round 6,
    tools/host_profile.py ddp: 3.0 ms of host time per step).  dev=None: the current device."""
    if _raw_stream is None:
        return torch.cuda.current_stream(dev)
    idx = _raw_device() if (dev is None or dev.index is None) else dev.index
    key = (idx, _raw_stream(idx))          # (the default stream has handle 0 on EVERY device)
    s = _STREAM_OBJ.get(key)
    if s is None:
        s = _STREAM_OBJ[key] = torch.cuda.current_stream(idx)
    return s


def _wg_fork(weight, wanted=True):
    """Called at the top of a convolution's backward node: returns the token for _wg_section (an event recorded on the current stream
    BEFORE the data gradient is enqueued, so the weight gradient may start beside it), or None when the weight gradient stays on the
    caller's stream (switch off, CPU, stream capture, or the parameter already holds a .grad: AccumulateGrad would then add on the
    caller's stream what the other stream is still writing)."""
    from . import config
    if not (wanted and config.wgrad_stream() and weight.is_cuda and weight.grad is None) or not config.side_streams_allowed():
        return None
    from . import streams
    dev = weight.device
    cur = _current_stream_object(dev)
    wg = streams.side_stream(dev, cur, streams.ROLE_WGRAD)      # (a high-priority stream here: 25.4 -> 38 ms per step)
    if wg == cur:
        return None
    ev = torch.cuda.Event()
    ev.record(cur)
    return ev, cur, wg


class _wg_section:
    """with _wg_section(token, inputs) as sec: <weight-gradient launches>; sec.publish(gw, gb).  `inputs`: the tensors those launches
    read (they were allocated on other streams and may be freed by autograd as soon as the node returns).  publish(): the results were
    allocated on the weight-gradient stream and will be read on the caller's."""

    def __init__(self, token, inputs):
        self.token, self.inputs, self.ctx = token, inputs, None

    def __enter__(self):
        if self.token is not None:
            ev, cur, wg = self.token
            wg.wait_event(ev)
            torch.cuda.set_stream(wg)          # (the context manager costs 20 us per use)
        return self

    def __exit__(self, *exc):
        if self.token is not None:
            ev, cur, wg = self.token
            torch.cuda.set_stream(cur)
            for t in self.inputs:
                if t is not None:
                    t.record_stream(wg)
            _WG["dirty"][wg.cuda_stream] = wg
            if not _WG["queued"]:
                _WG["queued"] = True
                torch.autograd.Variable._execution_engine.queue_callback(join_wgrad_stream)
        return False

    def publish(self, *outs):
        if self.token is not None:
            for t in outs:
                if t is not None:
                    t.record_stream(self.token[1])


def join_wgrad_stream():
    """Make the current stream wait for the weight gradients launched on the weight-gradient stream so far (config.set_wgrad_stream).
    Runs as an autograd-engine callback at the end of every backward pass that used the stream, in FusedAdam.step() and before the
    data-parallel reducer packs / exchanges a bucket; call it yourself before reading a .grad from inside a hook."""
    _WG["queued"] = False
    if _WG["dirty"]:
        for idx, wg in list(_WG["dirty"].items()):
            _current_stream_object(wg.device).wait_stream(wg)
        _WG["dirty"].clear()


# ------------------------------------------------------------------------------------------------ convolution
class Conv3d(torch.autograd.Function):
    """nn.Conv3d forward / data-gradient / weight-gradient (c3d.py:16, blocks_MDUNet.py:68,102,146)."""

    @staticmethod
    def forward(ctx, x, weight, bias, stride, pad, dil, want_stats=False, bias_grad_zero=False):
        _chk_dev(x, weight)
        ctx.set_materialize_grads(False)      # (the statistics output never has a gradient: no zero tensor of its shape per backward node)
        x = as_rows(x)
        rows, cx, ldx = rows_ld(x)
        N, Di, Hi, Wi = x.shape[:4]
        cout, cin, k = weight.shape[0], weight.shape[1], weight.shape[2]
        if cx < cin:
            raise ValueError(f"conv3d: input has {cx} channels, weight expects {cin}")
        Do, Ho, Wo = [(s + 2 * pad - dil * (k - 1) - 1) // stride + 1 for s in (Di, Hi, Wi)]
        y = torch.empty((N, Do, Ho, Wo, cout), dtype=x.dtype, device=x.device)
        b32 = None if bias is None else bias.detach()
        te = _tiled_elems(cin, cout, k, stride, pad, dil, Wi) if k > 1 else 0
        part = None
        if te:
            wq = _pack_conv_tiled(weight, 0, x.dtype, te, Wi)
            nblk = _lib.lib().dp_conv3d_tiled_stat_blocks(N, Di, Hi, Wi, cin, cout, k, cout, _dt(x)) if want_stats else 0
            if nblk:
                # the statistics of the normalisation that follows come out of the convolution's epilogue (values as stored)
                part = torch.empty((N, nblk, 2, cout), dtype=torch.float32, device=x.device)
                _lib.call("dp_conv3d_tiled_stats", _p(x), ldx, 0, 0, 0, _p(wq), _p(b32), _p(y), cout, _p(_tiled_ws(x, N, Di, Hi, Wi, cin, cout, k)),
                          _p(part), N, Di, Hi, Wi, cin, cout, k, _dt(x), _stream())
            else:
                _lib.call("dp_conv3d_tiled", _p(x), ldx, _p(wq), _p(b32), _p(y), cout, _p(_tiled_ws(x, N, Di, Hi, Wi, cin, cout, k)),
                          N, Di, Hi, Wi, cin, cout, k, _dt(x), _stream())
        elif k == 1 and stride == 1 and pad == 0:
            wp = _pack_conv(weight, 0, x.dtype)
            gemm_nt(x, wp, y, bias=b32, M=rows, N=cout, K=cin, lda=ldx, ldb=wp.shape[-1], ldc=cout, x3_terms=_x3_terms(True))
        elif N * Do * Ho * Wo <= 16384 and cin >= 32 and N * Do * Ho * Wo * k ** 3 * cin <= (1 << 26):
            # few output voxels, many channels (deep C3D stages): gather once, then ONE GEMM with K = taps * Cin
            wp = _pack_conv(weight, 0, x.dtype)                  # [Cout][tap][CinP]
            orow, kk = N * Do * Ho * Wo, wp.shape[1] * wp.shape[2]
            col = torch.empty((orow, kk), dtype=x.dtype, device=x.device)
            _lib.call("dp_im2col3d", _p(x), ldx, _p(col), N, Di, Hi, Wi, Do, Ho, Wo, cin, k, stride, pad, dil, _dt(x), _stream())
            gemm_nt(col, wp, y, bias=b32, M=orow, N=cout, K=kk, lda=kk, ldb=kk, ldc=cout)
        else:
            wp = _pack_conv(weight, 0, x.dtype)
            _lib.call("dp_conv3d", _p(x), ldx, _p(wp), _p(b32), _p(y), cout, N, Di, Hi, Wi, Do, Ho, Wo, cin, cout,
                      k, stride, pad, dil, 0, _dt(x), _stream())
        ctx.save_for_backward(x, weight)
        ctx.cfg = (stride, pad, dil, bias is not None)
        ctx.bias_grad_zero = bias_grad_zero
        ctx.bias_ref = bias if bias_grad_zero else None
        if want_stats:
            if part is None:
                part = _stats_partial(y)
            ctx.mark_non_differentiable(part)
            return y, part
        return y

    @staticmethod
    def backward(ctx, gy, *unused):
        if gy is None:
            return (None,) * 8
        x, weight = ctx.saved_tensors
        stride, pad, dil, has_bias = ctx.cfg
        gy = as_rows(gy)
        grows, cout, ldg = rows_ld(gy)
        rows, cx, ldx = rows_ld(x)
        N, Di, Hi, Wi = x.shape[:4]
        Do, Ho, Wo = gy.shape[1:4]
        cin, k = weight.shape[1], weight.shape[2]
        dtc = _dt(x)
        gx = gw = gb = None
        tok = _wg_fork(weight, ctx.needs_input_grad[1])
        if ctx.needs_input_grad[0]:
            gx = torch.empty((N, Di, Hi, Wi, cx), dtype=x.dtype, device=x.device)
            if cx > cin:
                gx.zero_()
            if k == 1 and stride == 1 and pad == 0:
                wt = _pack_conv(weight, 1, x.dtype)          # [Cin][1][CoutP]
                gemm_nt(gy, wt, gx, M=grows, N=cin, K=cout, lda=ldg, ldb=wt.shape[-1], ldc=cx, x3_terms=_x3_terms(False))
            elif stride == 1 and _tiled_elems(cout, cin, k, 1, dil * (k - 1) - pad, dil, Wo):
                te = _tiled_elems(cout, cin, k, 1, dil * (k - 1) - pad, dil, Wo)
                wq = _pack_conv_tiled(weight, 1, x.dtype, te, Wo)
                _lib.call("dp_conv3d_tiled", _p(gy), ldg, _p(wq), 0, _p(gx), cx, _p(_tiled_ws(x, N, Do, Ho, Wo, cout, cin, k)),
                          N, Do, Ho, Wo, cout, cin, k, dtc, _stream())
            elif stride == 1:
                wt = _pack_conv(weight, 2, x.dtype)          # transposed + flipped: data gradient as a forward conv
                _lib.call("dp_conv3d", _p(gy), ldg, _p(wt), 0, _p(gx), cx, N, Do, Ho, Wo, Di, Hi, Wi, cout, cin,
                          k, 1, dil * (k - 1) - pad, dil, 0, dtc, _stream())
            else:
                wt = _pack_conv(weight, 1, x.dtype)
                _lib.call("dp_conv3d", _p(gy), ldg, _p(wt), 0, _p(gx), cx, N, Do, Ho, Wo, Di, Hi, Wi, cout, cin,
                          k, stride, pad, dil, 1, dtc, _stream())
        with _wg_section(tok, (x, gy)) as sec:
            gw, gb = Conv3d._weight_gradients(ctx, x, weight, gy, (N, Di, Hi, Wi, Do, Ho, Wo), (grows, cout, ldg, rows, cx, ldx, cin, k, dtc))
            sec.publish(gw, gb)
        return gx, gw, gb, None, None, None, None, None

    @staticmethod
    def _weight_gradients(ctx, x, weight, gy, dims, g):
        N, Di, Hi, Wi, Do, Ho, Wo = dims
        grows, cout, ldg, rows, cx, ldx, cin, k, dtc = g
        stride, pad, dil, has_bias = ctx.cfg
        gw = gb = None
        wse = _lib.lib().dp_pointwise_wgrad_ws_elems(grows, cin, cout) if (
            k == 1 and stride == 1 and pad == 0 and ctx.needs_input_grad[1] and grows >= 32768 and cout * cin <= 256) else 0
        if wse:
            # heads: a handful of channels over millions of voxels -> one HBM row stream gives dW and db together
            gw = _wgrad_buffer(weight, False)
            want_b = has_bias and ctx.needs_input_grad[2] and not ctx.bias_grad_zero
            gb = torch.empty((cout,), dtype=torch.float32, device=x.device) if want_b else None
            ws = torch.empty((wse,), dtype=torch.float32, device=x.device)
            _lib.call("dp_pointwise_wgrad_rows", _p(x), ldx, _p(gy), ldg, _p(gw), cin, _p(gb), _p(ws), grows, cin, cout, dtc, _stream())
            if has_bias and ctx.needs_input_grad[2] and ctx.bias_grad_zero:
                gb = _zero_bias_grad(ctx.bias_ref)
            return gw, gb
        if ctx.needs_input_grad[1] and k == 1 and stride == 1 and pad == 0 and grows < 32768:
            # pointwise conv over few voxels: dW[co][ci] = gy^T x, both k-major in memory (split over K to fill the chip)
            tiles = -(-cout // 64) * -(-cin // 64)
            sk = max(1, min(grows // 512, 256 // tiles))
            gw = _wgrad_buffer(weight, sk > 1)
            _lib.call("dp_gemm_tn", _p(gy), ldg, _p(x), ldx, _p(gw), cin, cout, cin, grows, sk, dtc, _stream())
        elif ctx.needs_input_grad[1]:
            taps = k * k * k
            wse = 0
            if USE_TILED and (k > 1 or grows >= 32768):
                wse = _lib.lib().dp_conv3d_wgrad_tiled_ws_elems(cin, cout, k, stride, pad, dil, 1, Wo)
            # the tiled kernel overwrites dW; the generic one accumulates into it
            gw = _wgrad_buffer(weight, not wse)
            if wse:
                ws = _zero_scratch(x.device, wse)
                wdt = dtc
                if k == 1 and dtc == 0 and _p(x) % 16 == 0 and _p(gy) % 16 == 0:
                    # fp32x3 with one-product weight gradients (config.set_x3_wgrad_terms(1), the default): the mixers' dW = x_hi gy_hi on the
                    # streaming row kernel, fp32 rows rounded to bf16 in registers (the exact-fp32 tiled kernel took 0.4-0.5 ms at 2 x 128^3)
                    from . import config
                    if config.x3() and config.x3_wgrad_terms() == 1 and _lib.lib().dp_conv3d_wgrad_rows_ok(ldx, ldg, grows, cin, cout, DP_X1):
                        wdt = DP_X1
                _lib.call("dp_conv3d_wgrad_tiled", _p(x), ldx, _p(gy), ldg, _p(gw), _p(ws), N, Di, Hi, Wi, cin, cout, k,
                          cin * taps, taps, 1, wdt, _stream())
            else:
                wgrad(x, ldx, gy, ldg, gw, (N, Di, Hi, Wi, Do, Ho, Wo), cin, cout, k, stride, pad, dil, 1, 0,
                      cin * taps, taps, 1, dtc)
        if has_bias and ctx.needs_input_grad[2]:
            if ctx.bias_grad_zero:
                # the output feeds a normalisation over batch statistics: sum_v d(loss)/dy[v][c] is identically zero (the reference
                # accumulates pure round-off there), so no column-sum pass over gy is made
                gb = _zero_bias_grad(ctx.bias_ref)
            else:
                gb = torch.empty((cout,), dtype=torch.float32, device=x.device)
                colsum_into(_p(gy), ldg, grows, cout, gb, dtc)
        return gw, gb


def _stats_partial(y):
    """Per-block (sum, sum of squares) rows of an NDHWC tensor: [N, nblk, 2, C] fp32 (dp_stats_partial)."""
    y = as_rows(y)
    rows, C, ld = rows_ld(y)
    N = y.shape[0]
    V = rows // N
    part = torch.empty((N, _lib.lib().dp_stats_nblk(V), 2, C), dtype=torch.float32, device=y.device)
    _lib.call("dp_stats_partial", _p(y), ld, N, V, C, _p(part), _dt(y), _stream())
    return part


def conv3d(x, weight, bias=None, stride=1, pad=0, dil=1, stats=False, bias_grad_zero=False):
    """stats=True: returns (y, part) where part [N, nblk, 2, Cout] are the partial normalisation statistics of y (taken from the
    convolution's epilogue when the tiled kernel runs -- accumulators rounded to the storage type, i.e. the statistics of y as stored --
    otherwise by a statistics pass): hand it to norm_act(..., stats=part).
    bias_grad_zero=True: the caller normalises y over batch statistics next (InstanceNorm, or BatchNorm in training mode), which
    makes the bias gradient identically zero: it is returned as exact zeros instead of a column sum of round-off."""
    if isinstance(x, (tuple, list)):
        return conv3d_cat(x[0], x[1], weight, bias, stride, pad, dil, stats, bias_grad_zero)
    if _x3_conv_ok(x, None, weight, stride, pad, dil):
        return _x3_conv_call(x, None, weight, bias, stats, bias_grad_zero)
    if stats or bias_grad_zero:
        return Conv3d.apply(x, weight, bias, stride, pad, dil, stats, bias_grad_zero)
    return Conv3d.apply(x, weight, bias, stride, pad, dil)


class Conv3dCat(torch.autograd.Function):
    """nn.Conv3d applied to torch.cat((xa, xb), dim=channels) WITHOUT materialising the concatenation ("virtual concat",
    dp_conv3d_tiled2 / dp_conv3d_wgrad_tiled2): reference call sites base_blocks.py:139-140, c3d.py:103-113.
    Only built by conv3d_cat() for shapes the tiled kernels support (k in {3,7}, stride 1, "same" padding)."""

    @staticmethod
    def forward(ctx, xa, xb, weight, bias, pad, want_stats=False, bias_grad_zero=False):
        _chk_dev(xa, xb, weight)
        ctx.set_materialize_grads(False)      # (the statistics output never has a gradient: no zero tensor of its shape per backward node)
        xa, xb = as_rows(xa), as_rows(xb)
        _, ca, lda = rows_ld(xa)
        _, cbp, ldb = rows_ld(xb)
        N, D, H, W = xa.shape[:4]
        cout, cin, k = weight.shape[0], weight.shape[1], weight.shape[2]
        y = torch.empty((N, D, H, W, cout), dtype=xa.dtype, device=xa.device)
        wq = _pack_conv_tiled(weight, 0, xa.dtype, _tiled_elems(cin, cout, k, 1, pad, 1, W), W)
        b32 = None if bias is None else bias.detach()
        nblk = _lib.lib().dp_conv3d_tiled_stat_blocks(N, D, H, W, cin, cout, k, cout, _dt(xa)) if want_stats else 0
        part = None
        if nblk:
            part = torch.empty((N, nblk, 2, cout), dtype=torch.float32, device=xa.device)
            _lib.call("dp_conv3d_tiled_stats", _p(xa), lda, _p(xb), ldb, ca, _p(wq), _p(b32), _p(y), cout,
                      _p(_tiled_ws(xa, N, D, H, W, cin, cout, k)), _p(part), N, D, H, W, cin, cout, k, _dt(xa), _stream())
        else:
            _lib.call("dp_conv3d_tiled2", _p(xa), lda, _p(xb), ldb, ca, _p(wq), _p(b32), _p(y), cout, 0, 0, 0,
                      _p(_tiled_ws(xa, N, D, H, W, cin, cout, k)), N, D, H, W, cin, cout, k, _dt(xa), _stream())
        ctx.save_for_backward(xa, xb, weight)
        ctx.cfg = (pad, bias is not None)
        ctx.bias_grad_zero = bias_grad_zero
        ctx.bias_ref = bias if bias_grad_zero else None
        if want_stats:
            if part is None:
                part = _stats_partial(y)
            ctx.mark_non_differentiable(part)
            return y, part
        return y

    @staticmethod
    def backward(ctx, gy, *unused):
        if gy is None:
            return (None,) * 7
        xa, xb, weight = ctx.saved_tensors
        pad, has_bias = ctx.cfg
        gy = as_rows(gy)
        grows, cout, ldg = rows_ld(gy)
        _, ca, lda = rows_ld(xa)
        _, cbp, ldb = rows_ld(xb)
        N, D, H, W = xa.shape[:4]
        cin, k = weight.shape[1], weight.shape[2]
        dtc = _dt(xa)
        gxa = gxb = gw = gb = None
        tok = _wg_fork(weight, ctx.needs_input_grad[2])
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            gxa = torch.empty((N, D, H, W, ca), dtype=xa.dtype, device=xa.device)
            gxb = torch.empty((N, D, H, W, cbp), dtype=xa.dtype, device=xa.device)
            if cbp > cin - ca:
                gxb.zero_()
            wq = _pack_conv_tiled(weight, 1, xa.dtype, _tiled_elems(cout, cin, k, 1, k - 1 - pad, 1, W), W)
            _lib.call("dp_conv3d_tiled2", _p(gy), ldg, 0, 0, 0, _p(wq), 0, _p(gxa), ca, _p(gxb), cbp, ca,
                      _p(_tiled_ws(xa, N, D, H, W, cout, cin, k)), N, D, H, W, cout, cin, k, dtc, _stream())
        with _wg_section(tok, (xa, xb, gy)) as sec:
            if ctx.needs_input_grad[2]:
                gw = _wgrad_buffer(weight, False)      # overwritten by the tiled kernel
                taps = k * k * k
                ws = _zero_scratch(xa.device, max(taps * cin * cout, _lib.lib().dp_conv3d_wgrad_tiled_ws_elems(cin, cout, k, 1, k // 2, 1, 1, W)))
                _lib.call("dp_conv3d_wgrad_tiled2", _p(xa), lda, _p(xb), ldb, ca, _p(gy), ldg, _p(gw), _p(ws), N, D, H, W, cin, cout, k,
                          cin * taps, taps, 1, dtc, _stream())
            if has_bias and ctx.needs_input_grad[3]:
                if ctx.bias_grad_zero:
                    gb = _zero_bias_grad(ctx.bias_ref)
                else:
                    gb = torch.empty((cout,), dtype=torch.float32, device=xa.device)
                    colsum_into(_p(gy), ldg, grows, cout, gb, dtc)
            sec.publish(gw, gb)
        return gxa, gxb, gw, gb, None, None, None


def conv3d_cat(xa, xb, weight, bias=None, stride=1, pad=0, dil=1, stats=False, bias_grad_zero=False):
    """conv3d(cat((xa, xb), channels)): virtual concat when the tiled kernels support the shape, else a real cat."""
    cout, cin, k = weight.shape[0], weight.shape[1], weight.shape[2]
    ca, W = xa.shape[-1], xa.shape[3]
    if _x3_conv_ok(xa, xb, weight, stride, pad, dil):
        return _x3_conv_call(xa, xb, weight, bias, stats, bias_grad_zero)
    ok = (USE_TILED and k > 1 and stride == 1 and dil == 1 and pad == k // 2 and ca % 8 == 0 and 0 < ca < cin
          and xb.shape[-1] >= cin - ca and xa.dtype == xb.dtype and tuple(xa.shape[:4]) == tuple(xb.shape[:4]))
    if ok:
        L = _lib.lib()
        ok = bool(_tiled_elems(cin, cout, k, 1, pad, 1, W)) and bool(_tiled_elems(cout, cin, k, 1, k - 1 - pad, 1, W)) and \
            bool(L.dp_conv3d_wgrad_tiled_ws_elems(cin, cout, k, 1, pad, 1, 1, W))
    if not ok:
        return conv3d(cat((xa, xb)), weight, bias, stride, pad, dil, stats, bias_grad_zero)
    if stats or bias_grad_zero:
        return Conv3dCat.apply(xa, xb, weight, bias, pad, stats, bias_grad_zero)
    return Conv3dCat.apply(xa, xb, weight, bias, pad)


class ConvTranspose2x(torch.autograd.Function):
    """nn.ConvTranspose3d(kernel 2, stride 2, bias=False) (base_blocks.py:118-127; MONAI UnetrPrUpBlock):
    GEMM [voxels x Cin] x [Cin x 8 Cout] then a 2x2x2 pixel shuffle."""

    @staticmethod
    def forward(ctx, x, weight):
        _chk_dev(x, weight)
        x = as_rows(x)
        rows, cx, ldx = rows_ld(x)
        N, D, H, W = x.shape[:4]
        cin, cout = weight.shape[0], weight.shape[1]
        wp = _pack_tconv(weight, False, x.dtype)
        y = torch.empty((N, 2 * D, 2 * H, 2 * W, cout), dtype=x.dtype, device=x.device)
        # one launch where the matrix-core row kernel takes the shape (the pixel shuffle is its store pattern) ...
        rc = 3
        if rows >= 32768 and (x.dtype != torch.float32 or _x3_terms(True)):
            rc = _lib.call("dp_tconv2x_fwd", _p(x), ldx, _p(wp), wp.shape[-1], _p(y), cout, N, D, H, W, cin, cout,
                           DP_X3 if x.dtype == torch.float32 else _dt(x), _stream())
        if rc == 3:
            # ... else the GEMM into a [voxels][8 Cout] intermediate and the shuffle pass
            tmp = torch.empty((rows, 8 * cout), dtype=x.dtype, device=x.device)
            gemm_nt(x, wp, tmp, M=rows, N=8 * cout, K=cin, lda=ldx, ldb=wp.shape[-1], ldc=8 * cout)
            _lib.call("dp_pixel_shuffle2", _p(tmp), _p(y), N, D, H, W, cout, cout, _dt(x), _stream())
        ctx.save_for_backward(x, weight)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight = ctx.saved_tensors
        gy = as_rows(gy)
        _, cout, ldg = rows_ld(gy)
        rows, cx, ldx = rows_ld(x)
        N, D, H, W = x.shape[:4]
        cin = weight.shape[0]
        dtc = _dt(x)
        gu = torch.empty((rows, 8 * cout), dtype=x.dtype, device=x.device)
        _lib.call("dp_pixel_unshuffle2", _p(gy), ldg, _p(gu), N, D, H, W, cout, dtc, _stream())
        gx = gw = None
        if ctx.needs_input_grad[0]:
            wt = _pack_tconv(weight, True, x.dtype)          # [Cin][(abc,co)P]
            gx = torch.empty((N, D, H, W, cx), dtype=x.dtype, device=x.device)
            if cx > cin:
                gx.zero_()
            gemm_nt(gu, wt, gx, M=rows, N=cin, K=8 * cout, lda=8 * cout, ldb=wt.shape[-1], ldc=cx, x3_terms=_x3_terms(False))
        if ctx.needs_input_grad[1]:
            wse = _lib.lib().dp_conv3d_wgrad_tiled_ws_elems(cin, 8 * cout, 1, 1, 0, 1, 1, W) if (USE_TILED and rows >= 32768) else 0
            if wse:
                # ONE pointwise weight gradient with 8*Cout "output channels" (column (abc, co) of the unshuffled gradient):
                # x is read once instead of 8 times; the small fp32 result [(abc,co)][ci] is permuted into torch's [ci][co][abc]
                ws = _zero_scratch(x.device, wse)
                tmp = torch.empty((8 * cout, cin), dtype=torch.float32, device=x.device)
                _lib.call("dp_conv3d_wgrad_tiled", _p(x), ldx, _p(gu), 8 * cout, _p(tmp), _p(ws), N, D, H, W, cin, 8 * cout, 1,
                          cin, 1, 0, dtc, _stream())
                gw = tmp.view(8, cout, cin).permute(2, 1, 0).contiguous().view(weight.shape)
            elif rows <= 16384:
                # few voxels, many channels (the decoder's deep stages): dW^T[(abc,co)][ci] = gu^T x as a TN GEMM (k = voxel rows,
                # split so that the small output grid still fills the chip)
                tiles = -(-8 * cout // 64) * -(-cin // 64)
                sk = max(1, min(rows // 512, 512 // tiles))
                tmp = _pass_zeros((8 * cout, cin), x.device) if sk > 1 else torch.empty((8 * cout, cin), dtype=torch.float32, device=x.device)
                _lib.call("dp_gemm_tn", _p(gu), 8 * cout, _p(x), ldx, _p(tmp), cin, 8 * cout, cin, rows, sk, dtc, _stream())
                gw = tmp.view(8, cout, cin).permute(2, 1, 0).contiguous().view(weight.shape)
            else:
                # "tap" = abc selects the gy column block abc*Cout; x is not shifted
                gw = _wgrad_buffer(weight, True)   # [Cin][Cout][8]
                wgrad(x, ldx, gu, 8 * cout, gw, (1, 1, 1, rows, 1, 1, rows), cin, cout, 2, 1, 0, 1, 0, cout, 8, cout * 8, 1, dtc)
        return gx, gw


def conv_transpose2x(x, weight):
    return ConvTranspose2x.apply(x, weight)




# ------------------------------------------------------------------------------------------------ fp32x3 mode (csrc/x3.hip)
DP_X3 = 3
DP_X1 = 4
_PAT_ACT, _PAT_W = 0b010, 0b100      # operand blocks [hi | lo | hi] against [hi | hi | lo]: hi*hi + lo*hi + hi*lo


def _pack_one(w, dst, desc):
    """Build ONE packed copy through dp_pack_multi (a one-row table): the x3 layouts only exist as dp_pack_multi kinds."""
    L = _lib.lib()
    n = _pack_chunks(L, desc, dst, L.dp_pack_chunk())
    dev = w.device
    tab = torch.tensor([(w.data_ptr(), dst.data_ptr()) + tuple(desc)], dtype=torch.int64, device=dev)
    ct = torch.zeros((n,), dtype=torch.int32, device=dev)
    ci = torch.arange(n, dtype=torch.int32, device=dev)
    _lib.call("dp_pack_multi", _p(tab), _p(ct), _p(ci), n, _DT[dst.dtype], _stream())


def _x3_kind(base, pattern, cp):
    return base | (pattern << 8) | (cp << 16)


def _pack_conv_tiled_x3(w, tf, cp, W):
    """bf16 weights of an x3 convolution: role input channels [w_hi | w_hi | w_lo] over 3 * cp virtual channels (tf = 1: transposed +
    flipped, the data-gradient convolution, whose input channels are the layer's output channels)."""
    k = w.shape[2]
    co, ci = (w.shape[1], w.shape[0]) if tf else (w.shape[0], w.shape[1])
    L = _lib.lib()
    elems = L.dp_conv3d_tiled_weight_elems(3 * cp, co, k, 1, k // 2, 1, W)
    layout = L.dp_conv3d_tiled_layout(3 * cp, co, k, 1, k // 2, 1, W)
    if not elems:
        raise _lib.DoseHipError("x3 convolution: shape outside the tiled kernels")
    if layout == 2:
        desc = (_x3_kind(6, _PAT_W, cp), co, ci, k, 0, 1 if tf else 0)
    else:
        desc = (_x3_kind(4, _PAT_W, cp), co, ci, k, L.dp_conv3d_tiled_npair(co), 1 if tf else 0)

    def build():
        dst = torch.empty((elems,), dtype=torch.bfloat16, device=w.device)
        _pack_one(w.detach().contiguous(), dst, desc)
        return dst
    return _packs.get(w, ("conv_x3", tf, cp, elems, layout), build, lambda dst: desc)


def _pack_mat_x3(w, transposed, cp, pattern):
    """Linear weight [out][in] -> bf16 [out][3 cp] (cp >= in) or, transposed, [in][3 cp] (cp >= out), blocks per `pattern`."""
    nout, nin = w.shape
    rows = nin if transposed else nout
    desc = (_x3_kind(2, pattern, cp), nin, nout, 3 * cp, 0, 0) if transposed else (_x3_kind(1, pattern, cp), nout, nin, 3 * cp, 0, 0)

    def build():
        dst = torch.empty((rows, 3 * cp), dtype=torch.bfloat16, device=w.device)
        _pack_one(w.detach().contiguous(), dst, desc)
        return dst
    return _packs.get(w, ("mat_x3", transposed, cp, pattern), build, lambda dst: desc)


def split_rows(a, ca, b, cb, cp, parts, pattern):
    """fp32 rows cat(a[..., :ca], b[..., :cb]) -> bf16 [..., parts * cp] of hi / lo blocks (dp_split_rows)."""
    rows, _, lda = rows_ld(a)
    ldb = rows_ld(b)[2] if b is not None else 0
    out = torch.empty(tuple(a.shape[:-1]) + (parts * cp,), dtype=torch.bfloat16, device=a.device)
    _lib.call("dp_split_rows", _p(a), lda, ca, _p(b), ldb, cb, _p(out), cp, parts, pattern, rows, _stream())
    return out


def _x3_min_w(weight):
    """Shortest row the x3 convolution path takes: 8 -- the 12^3 level of the 96^3 crop (the cascade's no-grad OAR-TRANSEG windows, training
    at the reference's own crop size) fell to the exact-fp32 kernel at 2.4 ms per 7x7x7 launch, 24 ms of the 134-ms C5 step (round 5) --
    except with THREE-product weight gradients, whose tiled kernels start at 16."""
    if torch.is_grad_enabled() and weight.requires_grad:
        from . import config
        return 8 if config.x3_wgrad_terms() == 1 else 16        # (one-product weight gradients of short rows: the generic kernel on x_hi, gy_hi)
    return 8


def _x3_conv_shape_ok(W, cin, cout, k, stride, pad, dil, min_w=16):
    """Shape test of the x3 convolution path (ops.Conv3dX3) alone."""
    if not (USE_TILED and k in (3, 7) and stride == 1 and dil == 1 and pad == k // 2 and W >= min_w and cout >= 8 and cin >= 1):
        return False
    cp = (cin + 15) // 16 * 16
    return bool(_lib.lib().dp_conv3d_tiled_weight_elems(3 * cp, cout, k, 1, pad, 1, W))


_SPLIT_LAST = [None]


def _split_conv_input(xa, ca, xb, cb, cp):
    """split_rows for a convolution input, remembering the LAST result: the 3^3 and the 7^3 branch of a multi-scale block read the
    same (virtually concatenated) tensor one after the other (blocks_MDUNet.py:150-152) and share one split.  The entry is valid only
    while the very same tensor objects are alive and unmodified (weak references + version counters)."""
    import weakref
    key = (ca, cb, cp, xa.data_ptr(), xa._version, tuple(xa.shape), xa.stride(),
           None if xb is None else (xb.data_ptr(), xb._version, tuple(xb.shape), xb.stride()))
    ent = _SPLIT_LAST[0]
    if ent is not None and ent[0] == key and ent[1]() is xa and (xb is None or ent[2]() is xb):
        _SPLIT_LAST[0] = None             # (the pattern is exactly two consumers: do not keep half a gigabyte alive beyond the second)
        xs, ev, sh = ent[3], ent[4], ent[5]
        if sh != _stream():
            # the other branch runs on ANOTHER stream (config.set_branch_stream: the 3^3 branch beside the 7^3 one): wait for the split where
            # it was made instead of making it twice -- round 6: with the stream in the key every level's input was split once per branch,
            # 0.27 ms per 2 x 128^3 x 32-channel pair (tools/probes/x3_split_sites_probe.py)
            cur = _current_stream_object(xs.device)
            cur.wait_event(ev)
            xs.record_stream(cur)
        return xs
    xs = split_rows(xa, ca, xb, cb, cp, 2, 0b10)
    ev = torch.cuda.Event()
    ev.record(_current_stream_object(xs.device))
    _SPLIT_LAST[0] = (key, weakref.ref(xa), None if xb is None else weakref.ref(xb), xs, ev, _stream())
    return xs


def _x3_conv_ok(xa, xb, weight, stride, pad, dil):
    from . import config
    if not (config.x3() and USE_TILED and xa.is_cuda):
        return False
    cout, cin, k = weight.shape[0], weight.shape[1], weight.shape[2]
    W = xa.shape[3]
    if xa.dtype == torch.bfloat16:
        # an operand that already is split (norm_act(..., x3_split_for=...) wrote [x_hi | x_lo]): the producer checked the shape
        if xb is not None or xa.shape[-1] != 2 * cin or cin % 16 or not _x3_conv_shape_ok(W, cin, cout, k, stride, pad, dil, _x3_min_w(weight)):
            raise _lib.DoseHipError("conv3d: a bf16 tensor in the fp32x3 mode must be the [x_hi | x_lo] operand of an x3 convolution")
        return True
    if xa.dtype != torch.float32:
        return False
    if not (k in (3, 7) and stride == 1 and dil == 1 and pad == k // 2 and W >= _x3_min_w(weight) and cout >= 8):
        return False
    if xb is not None:
        ca = xa.shape[-1]
        if not (0 < ca < cin and xb.shape[-1] >= cin - ca and xb.dtype == xa.dtype and tuple(xa.shape[:4]) == tuple(xb.shape[:4])):
            return False
    elif xa.shape[-1] < cin:
        return False
    cp = (cin + 15) // 16 * 16
    return bool(_lib.lib().dp_conv3d_tiled_weight_elems(3 * cp, cout, k, 1, pad, 1, W))


# gradient tensors handed over in split form (NormAct.backward -> Conv3dX3.backward), keyed by address: a cheap handshake that the
# fp32-typed tensor arriving at the convolution really holds [gy_hi | gy_lo]
_GY_SPLIT_SENT = {}
_GY_SPLIT_CB = [False]
_PRESPLIT_OUT = {}            # split operands written by NormAct (by address) that no convolution has consumed yet


def _gy_split_reset():
    _GY_SPLIT_SENT.clear()
    _GY_SPLIT_CB[0] = False


class Conv3dX3(torch.autograd.Function):
    """nn.Conv3d (k in {3, 7}, stride 1, "same" padding) in the fp32x3 mode, on a tensor or on the virtual concatenation of two:
    fp32 tensors in HBM, the tuned bf16 MFMA kernels on split operands (csrc/x3.hip), fp32 results.  Forward and data gradient are
    ONE launch each over 3 x the (16-padded) channels; the weight gradient is two launches (x_hi | x_lo against gy_hi, x_hi against
    gy_lo) plus a small combine.  The split input is what is saved for the backward pass (same bytes as the fp32 tensor)."""

    @staticmethod
    def forward(ctx, xa, xb, weight, bias, want_stats=False, bias_grad_zero=False, gy_split=False):
        _chk_dev(xa, xb, weight)
        ctx.set_materialize_grads(False)      # (the statistics output never has a gradient: no zero tensor of its shape per backward node)
        xa = as_rows(xa)
        xb = None if xb is None else as_rows(xb)
        cout, cin, k = weight.shape[0], weight.shape[1], weight.shape[2]
        N, D, H, W = xa.shape[:4]
        ca = cin if xb is None else xa.shape[-1]
        cb = cin - ca
        cp = (cin + 15) // 16 * 16
        presplit = xa.dtype == torch.bfloat16
        if presplit:
            # written as [x_hi | x_lo] by the normalisation in front (NormAct).  Exactly ONE convolution may consume such a tensor: its
            # gradient travels back as fp32 data in a bf16-typed tensor, which autograd could not add to a second consumer's
            if not _PRESPLIT_OUT.pop(xa.data_ptr(), False):
                raise _lib.DoseHipError("conv3d (fp32x3): a split operand written by norm_act(..., x3_split_for=conv) has a second consumer")
            xs = xa.contiguous()
        else:
            xs = _split_conv_input(xa, ca, xb, cb, cp)                 # [.., x_hi (cp) | x_lo (cp)]
        # gy_split: a normalisation over this output follows (_x3_conv_call): its backward pass hands the gradient over ALREADY split
        # (dp_norm_act_bwd_apply_x3), disguised as an fp32 tensor of y's shape so that it can cross the autograd edge -- see NormAct
        wq = _pack_conv_tiled_x3(weight, 0, cp, W)
        y = torch.empty((N, D, H, W, cout), dtype=torch.float32, device=xa.device)
        b32 = None if bias is None else bias.detach()
        L = _lib.lib()
        nblk = L.dp_conv3d_tiled_stat_blocks(N, D, H, W, 3 * cp, cout, k, cout, DP_X3) if want_stats else 0
        ws = _tiled_ws(xa, N, D, H, W, 3 * cp, cout, k)
        part = None
        # a DP_X3 launch: Cin = 3 cp names the packed weights' contraction axis; the input is the 2 cp channel tensor [x_hi | x_lo], whose
        # x_hi chunks are staged once and swept against both their weight blocks
        if nblk:
            part = torch.empty((N, nblk, 2, cout), dtype=torch.float32, device=xa.device)
            _lib.call("dp_conv3d_tiled_stats", _p(xs), 2 * cp, 0, 0, 0, _p(wq), _p(b32), _p(y), cout, _p(ws), _p(part),
                      N, D, H, W, 3 * cp, cout, k, DP_X3, _stream())
        else:
            _lib.call("dp_conv3d_tiled2", _p(xs), 2 * cp, 0, 0, 0, _p(wq), _p(b32), _p(y), cout, 0, 0, 0, _p(ws),
                      N, D, H, W, 3 * cp, cout, k, DP_X3, _stream())
        ctx.save_for_backward(xs, weight)
        ctx.geom = (N, D, H, W, cin, cout, k, cp, ca, cin if presplit else xa.shape[-1], None if xb is None else xb.shape[-1])
        ctx.has_bias = bias is not None
        ctx.bias_grad_zero = bias_grad_zero
        ctx.bias_ref = bias if bias_grad_zero else None
        ctx.presplit, ctx.gy_split = presplit, gy_split
        if want_stats:
            if part is None:
                part = _stats_partial(y)
            ctx.mark_non_differentiable(part)
            return y, part
        return y

    @staticmethod
    def backward(ctx, gy, *unused):
        if gy is None:
            return (None,) * 7
        xs, weight = ctx.saved_tensors
        N, D, H, W, cin, cout, k, cp, ca, cxa, cxb = ctx.geom
        if ctx.gy_split:
            if not _GY_SPLIT_SENT.pop(gy.data_ptr(), False):
                raise _lib.DoseHipError("Conv3dX3: expected the split gradient of the normalisation that follows this convolution")
            gy = gy.contiguous()
        gy = as_rows(gy)
        grows, _, ldg = rows_ld(gy)
        dev = gy.device
        L = _lib.lib()
        pad, taps = k // 2, k * k * k
        cpo = (cout + 15) // 16 * 16
        need_x = ctx.needs_input_grad[0] or (cxb is not None and ctx.needs_input_grad[1])
        need_w = ctx.needs_input_grad[2]
        from . import config as _cfg
        one = _cfg.x3_dgrad_terms() == 1 and _tiled_elems(cout, cin, k, 1, pad, 1, W) > 0
        ldgs = 2 * cpo
        if ctx.gy_split:
            gys = gy.view(torch.bfloat16)                 # [.., gy_hi (cout) | gy_lo (cout)] already (cpo == cout)
        elif (one or not need_x) and (_cfg.x3_wgrad_terms() == 1 or not need_w):
            # one-product gradients on both sides: only gy_hi is ever read -- a compact bf16 tensor (half the bytes written here, and
            # the kernels' 32-byte rows are not interleaved with 32 bytes nobody wants)
            gys = split_rows(gy, cout, None, 0, cpo, 1, 0) if (need_x or need_w) else None
            ldgs = cpo
        else:
            gys = split_rows(gy, cout, None, 0, cpo, 2, 0b10) if (need_x or need_w) else None
        gxa = gxb = gw = gb = None
        tok = _wg_fork(weight, need_w)
        if need_x:
            if one or L.dp_conv3d_tiled_weight_elems(3 * cpo, cin, k, 1, pad, 1, W):
                if one:
                    # config.set_x3_dgrad_terms(1): gy_hi against the ordinary bf16 data-gradient pack, fp32 result (a DP_X1 launch)
                    wq = _pack_conv_tiled(weight, 1, torch.bfloat16, _tiled_elems(cout, cin, k, 1, pad, 1, W), W)
                    kc, kdt = cout, DP_X1
                else:
                    wq = _pack_conv_tiled_x3(weight, 1, cpo, W)
                    kc, kdt = 3 * cpo, DP_X3
                ws = _tiled_ws(gy, N, D, H, W, kc, cin, k)
                if cxb is None or ca % 8:
                    cx1 = cxa if cxb is None else cin            # (a concat split that is not a multiple of 8: one tensor, sliced below)
                    gx = torch.empty((N, D, H, W, cx1), dtype=torch.float32, device=dev)
                    if cx1 > cin:
                        gx.zero_()
                    _lib.call("dp_conv3d_tiled2", _p(gys), ldgs, 0, 0, 0, _p(wq), 0, _p(gx), cx1, 0, 0, 0, _p(ws),
                              N, D, H, W, kc, cin, k, kdt, _stream())
                    if cxb is None:
                        gxa = gx
                    else:
                        gxa = gx[..., :ca]
                        gxb = gx[..., ca:] if cxb == cin - ca else torch.cat((gx[..., ca:], gx.new_zeros((N, D, H, W, cxb - (cin - ca)))), -1)
                else:
                    gxa = torch.empty((N, D, H, W, ca), dtype=torch.float32, device=dev)
                    gxb = torch.empty((N, D, H, W, cxb), dtype=torch.float32, device=dev)
                    if cxb > cin - ca:
                        gxb.zero_()
                    _lib.call("dp_conv3d_tiled2", _p(gys), ldgs, 0, 0, 0, _p(wq), 0, _p(gxa), ca, _p(gxb), cxb, ca, _p(ws),
                              N, D, H, W, kc, cin, k, kdt, _stream())
            else:
                # fewer than 8 input channels (no tiled kernel computes so narrow an output): the exact-fp32 gather kernel
                wt = _pack_conv(weight, 2, torch.float32)
                gx = torch.empty((N, D, H, W, cin), dtype=torch.float32, device=dev)
                _lib.call("dp_conv3d", _p(gy), ldg, _p(wt), 0, _p(gx), cin, N, D, H, W, D, H, W, cout, cin, k, 1, k - 1 - pad, 1, 0, 0, _stream())
                if cxb is None:
                    gxa = gx if cxa == cin else torch.cat((gx, gx.new_zeros((N, D, H, W, cxa - cin))), -1)
                else:
                    gxa = gx[..., :ca]
                    gxb = gx[..., ca:] if cxb == cin - ca else torch.cat((gx[..., ca:], gx.new_zeros((N, D, H, W, cxb - (cin - ca)))), -1)
        with _wg_section(tok, (xs, gys, gy)) as sec:
            if need_w:
                from . import config
                wse = max(L.dp_conv3d_wgrad_tiled_ws_elems(2 * cp, cout, k, 1, pad, 1, 1, W), L.dp_conv3d_wgrad_tiled_ws_elems(cp, cout, k, 1, pad, 1, 1, W))
                if not wse:
                    # (cannot happen for a shape _x3_conv_ok admitted: the tiled weight-gradient kernels take every row of >= 8 voxels and
                    # _x3_min_w is 8; the generic-kernel fallback that used to sit here was unreachable and untested)
                    raise _lib.DoseHipError("x3 convolution: weight gradient outside the tiled kernels")
                ws = _zero_scratch(dev, wse)
                gw = _wgrad_buffer(weight, False)
                if config.x3_wgrad_terms() == 1:
                    # (config.set_x3_wgrad_terms(1)) x_hi x gy_hi only: one bf16 launch straight into dW
                    _lib.call("dp_conv3d_wgrad_tiled", _p(xs), 2 * cp, _p(gys), ldgs, _p(gw), _p(ws), N, D, H, W, cin, cout, k,
                              cin * taps, taps, 1, 1, _stream())
                else:
                    # S[co][p cp + ci][tap]: blocks p = 0, 1 from (x_hi | x_lo) x gy_hi, block 2 from x_hi x gy_lo
                    S = torch.empty((cout, 3 * cp, taps), dtype=torch.float32, device=dev)
                    _lib.call("dp_conv3d_wgrad_tiled", _p(xs), 2 * cp, _p(gys), 2 * cpo, _p(S), _p(ws), N, D, H, W, 2 * cp, cout, k,
                              3 * cp * taps, taps, 1, 1, _stream())
                    _lib.call("dp_conv3d_wgrad_tiled", _p(xs), 2 * cp, gys.data_ptr() + 2 * cpo, 2 * cpo, S.data_ptr() + 4 * 2 * cp * taps, _p(ws),
                              N, D, H, W, cp, cout, k, 3 * cp * taps, taps, 1, 1, _stream())
                    _lib.call("dp_x3_wgrad_combine", _p(S), _p(gw), cout, cin, cp, taps, 3, _stream())
            if ctx.has_bias and ctx.needs_input_grad[3]:
                if ctx.bias_grad_zero:
                    gb = _zero_bias_grad(ctx.bias_ref)
                else:
                    gb = torch.empty((cout,), dtype=torch.float32, device=dev)
                    colsum_into(_p(gy), ldg, grows, cout, gb, 0)
            sec.publish(gw, gb)
        if ctx.presplit and gxa is not None:
            gxa = gxa.contiguous().view(torch.bfloat16)    # the input was a bf16 [.., 2 cin] tensor: same bytes, the producer (NormAct) reads it as fp32
        return gxa, gxb, gw, gb, None, None, None


def _x3_conv_call(xa, xb, weight, bias, stats, bias_grad_zero):
    """Conv3dX3 with the split-gradient handshake: when statistics are requested (a normalisation over y follows and is y's only
    consumer), the channel count is a multiple of 16 and no bias gradient has to be summed from gy, the partial-statistics tensor is
    tagged so that norm_act(y, ..., stats=part) returns its input gradient already split."""
    gy_split = bool(stats and weight.shape[0] % 16 == 0 and (bias is None or bias_grad_zero))
    if gy_split:
        #  fewer than 8 input channels: the data gradient falls back to the exact-fp32 gather kernel, which needs the real
        # fp32 gy -- the normalisation behind then hands its gradient over unsplit
        cout, cin, k = weight.shape[0], weight.shape[1], weight.shape[2]
        gy_split = bool(_lib.lib().dp_conv3d_tiled_weight_elems(3 * cout, cin, k, 1, k // 2, 1, xa.shape[3]))
    out = Conv3dX3.apply(xa, xb, weight, bias, stats, bias_grad_zero, gy_split)
    if stats:
        out[1]._dp_gy_split = gy_split
    return out


_X3_SEL = {}


def _x3_selector(n, dev):
    """bf16 vector (1, 0, 1, 1, 0, 1, ...) of length n (n % 3 == 0): block weights that turn the K-stacked [hi | hi | lo] rows of a
    gradient back into hi + lo."""
    key = (dev.type, dev.index, n)
    t = _X3_SEL.get(key)
    if t is None:
        if len(_X3_SEL) > 8:
            _X3_SEL.clear()
        t = _X3_SEL[key] = torch.tensor([1.0, 0.0, 1.0], dtype=torch.bfloat16, device=dev).repeat(n // 3)
    return t


class LinearX3(torch.autograd.Function):
    """nn.Linear on token rows in the fp32x3 mode: y = x' W'^T with x' = [x_hi | x_lo | x_hi] (one split pass) and the packed
    W' = [w_hi | w_hi | w_lo]: the bf16 NT GEMM over 3 K, fp32 output.  Backward: gy' = [gy_hi | gy_hi | gy_lo] serves the data
    gradient (against [w_hi | w_lo | w_hi] transposed) AND, read as 3 x rows of K-stacked operands next to the saved x', the weight
    gradient (grouped TN launch): sum_k gy'[k] x'[k] = gy_hi x_hi + gy_hi x_lo + gy_lo x_hi."""

    @staticmethod
    def forward(ctx, x, weight, bias, splitk, defer_wgrad=False, xs=None):
        """xs: the operand already split ([..., rows, 3 cp] bf16, blocks hi | lo | hi; x is then None and receives no gradient)."""
        nout, K = weight.shape
        if xs is None:
            _chk_dev(x, weight)
            x = as_rows(x)
            rows, _, ldx = rows_ld(x)
            cp = (K + 7) // 8 * 8
            xs = split_rows(x, K, None, 0, cp, 3, _PAT_ACT)
            xshape = tuple(x.shape)
        else:
            cp = xs.shape[-1] // 3
            rows = xs.numel() // (3 * cp)
            xshape = tuple(xs.shape[:-1]) + (K,)
            x = xs
        wp = _pack_mat_x3(weight, False, cp, _PAT_W)
        b32 = None if bias is None else bias.detach()
        from . import config as _cfg
        y = _gemm_nt_splitk_det(xs, wp, b32, rows, nout, 3 * cp, 3 * cp, 3 * cp, splitk) if (splitk > 1 and _cfg.deterministic(2)) else None
        if y is not None:
            y = y.view(xshape[:-1] + (nout,))
        else:
            y = (torch.zeros if splitk > 1 else torch.empty)(xshape[:-1] + (nout,), dtype=torch.float32, device=xs.device)
            gemm_nt(xs, wp, y, bias=b32, M=rows, N=nout, K=3 * cp, lda=3 * cp, ldb=3 * cp, ldc=nout, splitk=splitk)
        ctx.save_for_backward(xs, weight)
        ctx.geom = (xshape, rows, K, cp)
        ctx.has_bias = bias is not None
        ctx.bias_ref = bias if defer_wgrad else None
        ctx.defer = defer_wgrad
        return y

    @staticmethod
    def backward(ctx, gy):
        xs, weight = ctx.saved_tensors
        xshape, rows, K, cp = ctx.geom
        gy = as_rows(gy)
        _, nout, ldg = rows_ld(gy)
        cpo = (nout + 7) // 8 * 8
        dev = gy.device
        gx = gw = gb = None
        from . import config as _cfg
        d1 = _cfg.x3_dgrad_terms() == 1
        if (d1 or not ctx.needs_input_grad[0]) and (_cfg.x3_linear_wgrad_terms() == 1 or not ctx.needs_input_grad[1]):
            gys, ldgs = split_rows(gy, nout, None, 0, cpo, 1, 0), cpo   # one-product gradients on both sides: gy_hi alone, compact
        else:
            gys, ldgs = split_rows(gy, nout, None, 0, cpo, 3, _PAT_W), 3 * cpo             # [gy_hi | gy_hi | gy_lo]
        if ctx.needs_input_grad[0]:
            wt = _pack_mat_x3(weight, True, cpo, _PAT_ACT)             # [in][w_hi | w_lo | w_hi]
            gx = torch.empty(xshape, dtype=torch.float32, device=dev)
            # (config.set_x3_dgrad_terms(1): block 0 of both operands alone, gy_hi w_hi)
            gemm_nt(gys, wt, gx, M=rows, N=K, K=cpo if d1 else 3 * cpo, lda=ldgs, ldb=3 * cpo, ldc=K)
        want_b = ctx.has_bias and ctx.needs_input_grad[2]
        if ctx.needs_input_grad[1]:
            gw = _wgrad_buffer(weight, False)
            # K-stacked view: row (3 r + p) of the [3 rows][cp] matrix is block p of row r
            from . import config
            if config.x3_linear_wgrad_terms() == 1:
                # gy_hi x_hi only: block 0 of every row of both operands (row pitch 3 cp)
                if ctx.defer and _DEFER["enabled"] and rows <= 16384 and weight.grad is None and (not want_b or ctx.bias_ref.grad is None):
                    # (the bias gradient rides in the same problem: column sums of the gy_hi operand)
                    gb = torch.empty((nout,), dtype=torch.float32, device=dev) if want_b else None
                    _defer_wgrad(gys, ldgs, xs, 3 * cp, gw, gb, nout, K, rows)
                    want_b = False
                else:
                    _lib.call("dp_gemm_tn", _p(gys), ldgs, _p(xs), 3 * cp, _p(gw), K, nout, K, rows, 1, 1, _stream())
            elif (ctx.defer and _DEFER["enabled"] and rows <= 16384 and weight.grad is None and (not want_b or ctx.bias_ref.grad is None)):
                _defer_wgrad(gys, cpo, xs, cp, gw, None, nout, K, 3 * rows)
                if want_b:
                    # the bias gradient joins the grouped launch as one more (N = 1) problem: column sums of gy = gy''^T s with the
                    # K-stacked selector s = (1, 0, 1) per row: hi + lo of every row (the kernel's own column sum of the stacked
                    # operand would be 2 hi + lo)
                    gb = torch.empty((nout,), dtype=torch.float32, device=dev)
                    _defer_wgrad(gys, cpo, _x3_selector(3 * rows, dev), 1, gb, None, nout, 1, 3 * rows)
                    want_b = False
            else:
                tiles = -(-nout // 64) * -(-K // 64)
                sk = max(1, min(3 * rows // 512, 512 // tiles)) if tiles < 256 else 1
                if sk > 1:
                    gw.zero_()
                _lib.call("dp_gemm_tn", _p(gys), cpo, _p(xs), cp, _p(gw), K, nout, K, 3 * rows, sk, 1, _stream())
        if want_b:
            gb = torch.empty((nout,), dtype=torch.float32, device=dev)
            colsum_into(_p(gy), ldg, rows, nout, gb, 0)
        return gx, gw, gb, None, None, None


def patch_embed_x3(x, C, p, weight, bias, splitk):
    """fp32x3 patch embedding (MONAI PatchEmbeddingBlock 'perceptron': Rearrange + Linear) without an fp32 token matrix: the voxel
    tensor is split once ([x_hi | x_lo] per voxel) and each half is patchified straight into its column block(s) of the
    [hi | lo | hi] operand of the x3 GEMM (dp_patchify_ld).  Returns None when the shape is outside that kernel's fast path."""
    x = as_rows(x)
    _, cx, ld = rows_ld(x)
    B, S0, S1, S2 = x.shape[:4]
    K = p * p * p * C
    cpv = (C + 15) // 16 * 16
    if (K % 8 or weight.shape[1] != K or p * 2 * cpv > 1024 or p * C > 1024 or (p * C) % 8 or p * C * C >= (1 << 20) or S0 % p or S1 % p
            or S2 % p or x.dtype != torch.float32):
        return None
    # (the run kernel moves whole p-voxel runs of `ld` channels starting at the half it was pointed to: the x_lo pass reads cpv
    # elements past the last voxel row, so the split tensor gets one spare row)
    nvox = B * S0 * S1 * S2
    xv = torch.empty(((nvox + 1) * 2 * cpv,), dtype=torch.bfloat16, device=x.device)
    _lib.call("dp_split_rows", _p(x), ld, C, 0, 0, 0, _p(xv), cpv, 2, 0b10, nvox, _stream())
    ntok = (S0 // p) * (S1 // p) * (S2 // p)
    xs = torch.empty((B, ntok, 3 * K), dtype=torch.bfloat16, device=x.device)
    for blk, part in ((0, 0), (1, 1), (2, 0)):
        _lib.call("dp_patchify_ld", xv.data_ptr() + 2 * part * cpv, xs.data_ptr() + 2 * blk * K, 3 * K, B, S0, S1, S2, C, 2 * cpv, p, 1, _stream())
    return LinearX3.apply(None, weight, bias, splitk, True, xs)


# ------------------------------------------------------------------------------------------------ deferred weight gradients
# The weight / bias gradients of the transformer's Linear layers are 33 separate TN GEMMs + 25 column sums per step, each a
# latency-bound 5-25 us launch on 1024 token rows.  They feed nothing inside the backward pass, so a Linear created with
# defer_wgrad=True only RECORDS its (gy, x, dW, db) and returns the (still unwritten) gradient tensors; ONE grouped launch
# (dp_gemm_tn_grouped) fills all of them at the end of the backward pass, or earlier when somebody needs them (flush_deferred():
# the data-parallel reducer before it packs a bucket, FusedAdam.step()).
_DEFER = {"pending": [], "queued": False, "host": None, "rot": 0, "enabled": os.environ.get("DOSE_HIP_DEFER_WGRAD", "1") != "0"}


_TN_TILE128 = os.environ.get("DOSE_HIP_TN_TILE128", "1") != "0"


def _alias(t):
    """A second tensor object on t's storage that is NOT a view of t: holding it keeps the memory alive without raising t's own
    reference count, so AccumulateGrad still adopts t as .grad without a copy (it clones a gradient somebody else holds), and
    torch.autograd.grad() callers get t itself.  Whatever tensor ends up owning the storage sees what is written through the alias."""
    return torch.empty(0, dtype=t.dtype, device=t.device).set_(t.untyped_storage(), t.storage_offset(), t.shape, t.stride())


def _defer_wgrad(gy, ldg, x, ldx, gw, gb, nout, nin, rows):
    """Record one weight (+ bias) gradient for the grouped launch.  gw / gb are the still unwritten fp32 tensors the backward node is
    about to hand to autograd; aliases of them are recorded (recording the PARAMETERS and looking up p.grad at flush time
    left a window in which a parameter's hook had fired -- and the data-parallel reducer had exchanged its bucket -- while the entry
    was waiting for the partner's .grad, and leaked entries for ever under torch.autograd.grad)."""
    ev = torch.cuda.Event()
    ev.record()                                            # on the stream that produced gy (the ViT branch runs on a side stream)
    _DEFER["pending"].append((gy, ldg, x, ldx, _alias(gw), None if gb is None else _alias(gb), nout, nin, rows, ev, _current_stream_object()))
    if not _DEFER["queued"]:
        # (safety net: whatever is still pending at the end of the backward pass is flushed then)
        torch.autograd.Variable._execution_engine.queue_callback(flush_deferred)
        _DEFER["queued"] = True


def deferred_pending():
    """Number of recorded weight gradients that have not been launched yet (0 after flush_deferred())."""
    return len(_DEFER["pending"])


def flush_deferred(*_unused):
    """Launch the grouped weight-gradient GEMM for everything recorded so far, on the stream that recorded it (the ViT branch's side
    stream: the launch then overlaps the 128^3 branch's backward on the main stream), and make the current stream wait for it.
    EVERY recorded entry is launched (nothing is ever carried over to a later flush).  No-op when nothing is pending.  Also usable as
    a post-accumulate-grad hook (PatchEmbeddingBlock registers it on its weight: the first layer of the transformer is its last
    backward node)."""
    _DEFER["queued"] = False
    pend, _DEFER["pending"] = _DEFER["pending"], []
    cur = _current_stream_object() if (pend or _DEFER.get("last_stream") is not None) else None
    by = {}
    for e in pend:
        by.setdefault((e[0].dtype, e[0].device, e[10]), []).append(e)
    for (dtype, dev, st), lst in by.items():
        rows_tab, tile0 = [], 0
        for gy, ldg, x, ldx, gw, gb, nout, nin, rows, ev, _st in lst:
            if gw.dtype != torch.float32 or not gw.is_contiguous() or (gb is not None and not gb.is_contiguous()):
                raise _lib.DoseHipError("deferred weight gradient: the gradient tensor is not a contiguous fp32 tensor")
            # 128 x 128 tiles where they are whole and the rows aligned (half the L2 -> LDS operand traffic of 64 x 64 tiles)
            big = (_TN_TILE128 and nout % 128 == 0 and nin % 128 == 0 and ldg % 8 == 0 and ldx % 8 == 0 and gy.data_ptr() % 16 == 0
                   and x.data_ptr() % 16 == 0)
            ts = 128 if big else 64
            tm, tn = -(-nout // ts), -(-nin // ts)
            rows_tab.append((gy.data_ptr(), x.data_ptr(), gw.data_ptr(), 0 if gb is None else gb.data_ptr(), ldg, ldx, nin, nout, nin, rows, tile0,
                             tm | ((1 << 32) if big else 0)))
            tile0 += tm * tn
            for t in (gw, gb):
                if t is not None:
                    t.record_stream(st)
        # table: rotating pinned host buffers, each guarded by the event of the copy that last read it (the host thread runs several
        # steps ahead of the GPU when nothing synchronises: an unguarded buffer is overwritten before its copy has executed)
        n = len(rows_tab)
        if n == 0:
            continue
        if _DEFER["host"] is None or _DEFER["host"][0][0].shape[0] < n:
            for _h, e in (_DEFER["host"] or ()):
                if e is not None:
                    e.synchronize()
            # (64 slots: the data-parallel reducer flushes once per bucket, i.e. a dozen times per backward pass, and the host runs up to
            # a whole step ahead of the GPU -- with 4 slots the wait below blocked the launch thread on the GPU in the middle of
            # every backward pass: 4.9 ms of host time per step)
            _DEFER["host"] = [[torch.empty((max(n, 64), 12), dtype=torch.int64).pin_memory(), None] for _ in range(64)]
        slot = _DEFER["host"][_DEFER["rot"] % 64]
        _DEFER["rot"] += 1
        if slot[1] is not None and not torch.cuda.is_current_stream_capturing():     # (torch.cuda.graph synchronises on entry)
            slot[1].synchronize()
        host = slot[0]
        host[:n] = torch.tensor(rows_tab, dtype=torch.int64)
        with torch.cuda.stream(st):
            tab = torch.empty((n, 12), dtype=torch.int64, device=dev)
            tab.copy_(host[:n], non_blocking=True)
            slot[1] = None
            if not torch.cuda.is_current_stream_capturing():
                slot[1] = torch.cuda.Event()
                slot[1].record(st)
            _lib.call("dp_gemm_tn_grouped", _p(tab), n, tile0, _DT[dtype], st.cuda_stream)
        _DEFER["last_stream"] = st
    last = _DEFER.get("last_stream")
    if last is not None and cur is not None and last != cur:
        cur.wait_stream(last)           # whoever asked for the flush reads the gradients on the current stream
        if not pend:
            _DEFER["last_stream"] = None


class Linear(torch.autograd.Function):
    """nn.Linear on token rows (MONAI ViT blocks; patch embedding uses splitk)."""

    @staticmethod
    def forward(ctx, x, weight, bias, splitk, defer_wgrad=False):
        _chk_dev(x, weight)
        x = as_rows(x)
        rows, K, ldx = rows_ld(x)
        nout = weight.shape[0]
        wp = _pack_mat(weight, False, x.dtype)
        y = torch.empty(tuple(x.shape[:-1]) + (nout,), dtype=x.dtype, device=x.device)
        b32 = None if bias is None else bias.detach()
        if splitk > 1:
            from . import config as _cfg
            acc = _gemm_nt_splitk_det(x, wp, b32, rows, nout, K, ldx, wp.shape[-1], splitk) if _cfg.deterministic(2) else None
            if acc is None:
                acc = torch.zeros((rows, nout), dtype=torch.float32, device=x.device)
                gemm_nt(x, wp, acc, bias=b32, M=rows, N=nout, K=K, lda=ldx, ldb=wp.shape[-1], ldc=nout, splitk=splitk)
            if x.dtype == torch.float32:
                y = acc.view(y.shape)
            else:
                _lib.call("dp_cast", _p(acc), 0, _p(y), _dt(x), acc.numel(), _stream())
        else:
            gemm_nt(x, wp, y, bias=b32, M=rows, N=nout, K=K, lda=ldx, ldb=wp.shape[-1], ldc=nout)
        ctx.save_for_backward(x, weight)
        ctx.has_bias = bias is not None
        ctx.bias_ref = bias if defer_wgrad else None
        ctx.defer = defer_wgrad
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight = ctx.saved_tensors
        gy = as_rows(gy)
        rows, K, ldx = rows_ld(x)
        _, nout, ldg = rows_ld(gy)
        dtc = _dt(x)
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            wt = _pack_mat(weight, True, x.dtype)            # [in][outP]
            gx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            gemm_nt(gy, wt, gx, M=rows, N=K, K=nout, lda=ldg, ldb=wt.shape[-1], ldc=K)
        want_b = ctx.has_bias and ctx.needs_input_grad[2]
        if (ctx.defer and _DEFER["enabled"] and ctx.needs_input_grad[1] and rows <= 16384 and weight.grad is None
                and (not want_b or ctx.bias_ref.grad is None)):
            # recorded for the grouped launch at the end of the backward pass; dW and db are returned unwritten
            gw = _wgrad_buffer(weight, False)
            gb = torch.empty((nout,), dtype=torch.float32, device=x.device) if want_b else None
            _defer_wgrad(gy, ldg, x, ldx, gw, gb, nout, K, rows)
            return gx, gw, gb, None, None
        if ctx.needs_input_grad[1]:
            if rows <= 16384:
                # token matrices: dW[out][in] = gy^T x, both operands k-major (k = token rows) as they lie in memory
                gw = _wgrad_buffer(weight, False)
                _lib.call("dp_gemm_tn", _p(gy), ldg, _p(x), ldx, _p(gw), K, nout, K, rows, 1, dtc, _stream())
            else:
                gw = _wgrad_buffer(weight, True)
                wgrad(x, ldx, gy, ldg, gw, (1, 1, 1, rows, 1, 1, rows), K, nout, 1, 1, 0, 1, 0, 0, K, 1, 0, dtc)
        if ctx.has_bias and ctx.needs_input_grad[2]:
            gb = torch.empty((nout,), dtype=torch.float32, device=x.device)
            colsum_into(_p(gy), ldg, rows, nout, gb, dtc)
        return gx, gw, gb, None, None


_FUSED_MLP = os.environ.get("DOSE_HIP_FUSED_MLP", "1") != "0"      # (A/B switch for experiments)


class MLP(torch.autograd.Function):
    """MONAI MLPBlock, linear2(GELU(linear1(x))), as ONE autograd node: the GELU is the epilogue of linear1's GEMM and its derivative
    the epilogue of linear2's data-gradient GEMM (dp_gemm_nt_gelu), so neither the activation nor its gradient is a pass of its
    own; the four weight / bias gradients join the grouped launch (flush_deferred).  16-bit storage types (fp32: composed ops)."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2):
        _chk_dev(x, w1, w2)
        x = as_rows(x)
        rows, K, ldx = rows_ld(x)
        mid, nout = w1.shape[0], w2.shape[0]
        w1p, w2p = _pack_mat(w1, False, x.dtype), _pack_mat(w2, False, x.dtype)
        h = torch.empty(tuple(x.shape[:-1]) + (mid,), dtype=x.dtype, device=x.device)
        a = torch.empty_like(h)
        y = torch.empty(tuple(x.shape[:-1]) + (nout,), dtype=x.dtype, device=x.device)
        _lib.call("dp_gemm_nt_gelu", _p(x), ldx, _p(w1p), w1p.shape[-1], _p(a), mid, _p(b1.detach()), _p(h), mid, rows, mid, K, 1, _dt(x),
                  _stream())
        gemm_nt(a, w2p, y, bias=b2.detach(), M=rows, N=nout, K=mid, lda=mid, ldb=w2p.shape[-1], ldc=nout)
        ctx.save_for_backward(x, h, a, w1, w2)
        ctx.params = (w1, b1, w2, b2)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, h, a, w1, w2 = ctx.saved_tensors
        _, b1, _, b2 = ctx.params
        gy = as_rows(gy)
        rows, K, ldx = rows_ld(x)
        _, nout, ldg = rows_ld(gy)
        mid = w1.shape[0]
        dtc = _dt(x)
        # gh = (gy W2) * GELU'(h): the gradient with respect to linear1's output, in one GEMM
        w2t = _pack_mat(w2, True, x.dtype)                      # [mid][outP]
        gh = torch.empty_like(h)
        _lib.call("dp_gemm_nt_gelu", _p(gy), ldg, _p(w2t), w2t.shape[-1], _p(gh), mid, 0, _p(h), mid, rows, mid, nout, 2, dtc, _stream())
        gx = None
        if ctx.needs_input_grad[0]:
            w1t = _pack_mat(w1, True, x.dtype)                  # [in][midP]
            gx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            gemm_nt(gh, w1t, gx, M=rows, N=K, K=mid, lda=mid, ldb=w1t.shape[-1], ldc=K)
        grads = []
        for (w, b, g2, ldg2, inp, ldi, no, ni) in ((w1, b1, gh, mid, x, ldx, mid, K), (w2, b2, gy, ldg, a, mid, nout, mid)):
            if _DEFER["enabled"] and rows <= 16384 and w.grad is None and b.grad is None:
                gw = _wgrad_buffer(w, False)
                gb = torch.empty((no,), dtype=torch.float32, device=x.device)
                _defer_wgrad(g2, ldg2, inp, ldi, gw, gb, no, ni, rows)
            else:
                gw = _wgrad_buffer(w, False)
                _lib.call("dp_gemm_tn", _p(g2), ldg2, _p(inp), ldi, _p(gw), ni, no, ni, rows, 1, dtc, _stream())
                gb = torch.empty((no,), dtype=torch.float32, device=x.device)
                colsum_into(_p(g2), ldg2, rows, no, gb, dtc)
            grads += [gw, gb]
        return gx, grads[0], grads[1], grads[2], grads[3]


def mlp(x, w1, b1, w2, b2):
    """linear2(GELU(linear1(x))) (MONAI MLPBlock, dropout 0)."""
    if not _FUSED_MLP or x.dtype == torch.float32 or not (w1.requires_grad and w2.requires_grad and b1 is not None and b2 is not None
                                         and b1.requires_grad and b2.requires_grad) or x.shape[-1] % 8 or w1.shape[0] % 8 \
            or x.numel() // x.shape[-1] > 16384:
        return linear(gelu(linear(x, w1, b1, defer_wgrad=True)), w2, b2, defer_wgrad=True)
    return MLP.apply(x, w1, b1, w2, b2)


def linear(x, weight, bias=None, splitk=1, defer_wgrad=False):
    """defer_wgrad=True (weights that are used once per forward pass and not shared): the weight / bias gradients are produced by
    one grouped launch at the end of the backward pass instead of two to three small launches here."""
    from . import config
    if config.x3() and x.dtype == torch.float32 and x.is_cuda and x.shape[-1] >= 16 and weight.shape[0] >= 16:
        return LinearX3.apply(x, weight, bias, splitk, defer_wgrad)
    return Linear.apply(x, weight, bias, splitk, defer_wgrad)


# ------------------------------------------------------------------------------------------------ normalisation
def _norm_forward(x, kind, gamma, beta, running_mean, running_var, training, res, act, eps, momentum, y_ptr, ldy, apply=True, part=None,
                  split_cp=0):
    """Statistics + fused normalise/affine/residual/activation of one NDHWC tensor into (y_ptr, row pitch ldy).
    part: partial statistics rows [N, nblk, 2, C] already produced by the convolution that wrote x (conv3d(..., stats=True))."""
    rows, C, ldx = rows_ld(x)
    N = x.shape[0]
    V = rows // N
    L = _lib.lib()
    dtc = _dt(x)
    dev = x.device
    use_batch_stats = kind == "instance" or training
    own_rows = False
    if use_batch_stats:
        if part is not None:
            if tuple(part.shape[::2]) != (N, 2) or part.shape[3] != C:
                raise ValueError("norm_act: stats tensor does not belong to this input")
            nblk = part.shape[1]
        else:
            nblk = L.dp_stats_nblk(V)
            part = torch.empty((N, nblk, 2, C), dtype=torch.float32, device=dev)
            own_rows = True
        groups = N if kind == "instance" else 1
        mean = torch.empty((groups, C), dtype=torch.float32, device=dev)
        rstd = torch.empty((groups, C), dtype=torch.float32, device=dev)
        upd = kind == "batch" and training and running_mean is not None
        fin = (1 if kind == "batch" else 0, float(eps), _p(mean), _p(rstd), _p(running_mean) if upd else 0, _p(running_var) if upd else 0,
               float(momentum))
        # rows of our own: ONE launch, the last block of every statistics group finalizes it (3 = folded form off: the two calls)
        if not own_rows or _lib.call("dp_stats_partial_finalize", _p(x), ldx, N, V, C, _p(part), *fin, dtc, _stream()) == 3:
            if own_rows:
                _lib.call("dp_stats_partial", _p(x), ldx, N, V, C, _p(part), dtc, _stream())
            _lib.call("dp_stats_finalize", _p(part), N, nblk, C, V, *fin, _stream())
    else:   # eval-mode batch norm: running statistics
        mean = running_mean.detach().reshape(1, C).float()
        rstd = torch.empty((1, C), dtype=torch.float32, device=dev)
        zero_part = torch.zeros((1, 1, 2, C), dtype=torch.float32, device=dev)
        # rstd = 1/sqrt(var+eps) through the finalize kernel: feed sums s1=0, s2=var (count 1)
        zero_part[0, 0, 1].copy_(running_var.detach())
        dummy = torch.empty((1, C), dtype=torch.float32, device=dev)
        _lib.call("dp_stats_finalize", _p(zero_part), 1, 1, C, 1, 1, float(eps), _p(dummy), _p(rstd), 0, 0, 0.0, _stream())
    ssn = C if kind == "instance" else 0
    if not apply:       # statistics only (the caller normalises: norm_act_cat)
        return mean, rstd, use_batch_stats, ssn
    g32 = None if gamma is None else gamma.detach()
    b32 = None if beta is None else beta.detach()
    ldr = rows_ld(res)[2] if res is not None else 0
    if split_cp:
        _lib.call("dp_norm_act_fwd_x3", _p(x), ldx, _p(mean), _p(rstd), ssn, _p(g32), _p(b32), _p(res), ldr, _act_code(act, x.dtype),
                  y_ptr, split_cp, N, V, C, _stream())
    else:
        _lib.call("dp_norm_act_fwd", _p(x), ldx, _p(mean), _p(rstd), ssn, _p(g32), _p(b32), _p(res), ldr, _act_code(act, x.dtype),
                  y_ptr, ldy, N, V, C, dtc, _stream())
    return mean, rstd, use_batch_stats, ssn


def _norm_backward(x, mean, rstd, gamma, beta, res, kind, act, use_stats, ssn, gy_ptr, ldg, need_x, need_gb, need_res, split_cp=0):
    """Backward of _norm_forward for an upstream gradient at (gy_ptr, row pitch ldg) -> (gx, dgamma, dbeta, gres)."""
    rows, C, ldx = rows_ld(x)
    N = x.shape[0]
    V = rows // N
    L = _lib.lib()
    dtc = _dt(x)
    dev = x.device
    ldr = rows_ld(res)[2] if res is not None else 0
    g32 = None if gamma is None else gamma.detach()
    b32 = None if beta is None else beta.detach()
    nblk = L.dp_stats_nblk(V)
    groups = N if kind == "instance" else 1
    # ONE allocation for the pass's scratch -- [s1 | s2 | partial rows], handed to the kernels as pointers: three torch.empty calls cost the
    # launch thread ~8 us per normalisation (tools/host_profile.py: torch.empty is the largest single item of the host step)
    gc = groups * C
    scr = torch.empty((2 * gc + N * nblk * 2 * C,), dtype=torch.float32, device=dev)
    s1p = scr.data_ptr()
    s2p, partp = s1p + 4 * gc, s1p + 8 * gc
    # (dp_norm_bwd_finalize overwrites both in either mode: the sample-0 block of an instance normalisation combines every sample's rows)
    dgamma = torch.empty((C,), dtype=torch.float32, device=dev) if need_gb else None
    dbeta = torch.empty((C,), dtype=torch.float32, device=dev) if need_gb else None
    if use_stats or need_gb:
        src = (_p(x), ldx, gy_ptr, ldg, _p(mean), _p(rstd), ssn, _p(g32), _p(b32), _p(res), ldr, _act_code(act, x.dtype), N, V, C, partp)
        fin = (0 if kind == "instance" else 1, s1p, s2p, _p(dgamma), _p(dbeta))
        if _lib.call("dp_norm_act_bwd_partial_finalize", *src, *fin, dtc, _stream()) == 3:      # (3: folded form off / not applicable)
            _lib.call("dp_norm_act_bwd_partial", *src, dtc, _stream())
            _lib.call("dp_norm_bwd_finalize", partp, N, nblk, C, *fin, _stream())
    gx = gres = None
    if need_x or need_res:
        gres = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_res else None
        cnt = V if kind == "instance" else N * V
        if split_cp and need_x:
            gx = torch.empty(tuple(x.shape[:-1]) + (2 * split_cp,), dtype=torch.bfloat16, device=dev)      # [gx_hi | gx_lo]
            _lib.call("dp_norm_act_bwd_apply_x3", _p(x), ldx, gy_ptr, ldg, _p(mean), _p(rstd), ssn, _p(g32), _p(b32), _p(res), ldr,
                      _act_code(act, x.dtype), s1p, s2p, 1.0 / cnt, 1 if use_stats else 0, _p(gx), split_cp, _p(gres), C, N, V, C, _stream())
            return gx, dgamma, dbeta, gres
        gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        _lib.call("dp_norm_act_bwd_apply", _p(x), ldx, gy_ptr, ldg, _p(mean), _p(rstd), ssn, _p(g32), _p(b32), _p(res), ldr,
                  _act_code(act, x.dtype), s1p, s2p, 1.0 / cnt, 1 if use_stats else 0, _p(gx), C, _p(gres), C, N, V, C, dtc, _stream())
    return gx, dgamma, dbeta, gres


class NormAct(torch.autograd.Function):
    """InstanceNorm3d / BatchNorm3d (+affine) (+residual) + activation, fused.
    kind: 'instance' | 'batch'.  For 'batch', running buffers are updated in place when training."""

    @staticmethod
    def forward(ctx, x, kind, gamma, beta, running_mean, running_var, training, res, act, eps, momentum, stats=None, split_out=False,
                grad_split=False):
        """fp32x3 only -- split_out: y is written as the bf16 [y_hi | y_lo] operand of the x3 convolution that is its only consumer
        (shape [.., 2C]); grad_split: x is the output of an x3 convolution, whose backward pass takes the gradient in the same split
        form.  Both cross the autograd edge as a same-bytes reinterpretation: a bf16 [.., 2C] tensor and an fp32 [.., C] tensor are
        the same memory, so the gradient of a bf16 [.., 2C] output arrives as fp32 data viewed as bf16 (Conv3dX3 returns
        gx.view(bfloat16)), and the split gradient of an fp32 [.., C] input leaves as bf16 data viewed as fp32."""
        _chk_dev(x)
        x = as_rows(x)
        C = x.shape[-1]
        if res is not None:
            res = as_rows(res)
        if split_out:
            y = torch.empty(tuple(x.shape[:-1]) + (2 * C,), dtype=torch.bfloat16, device=x.device)
        else:
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean, rstd, use_batch_stats, ssn = _norm_forward(x, kind, gamma, beta, running_mean, running_var, training, res, act, eps,
                                                         momentum, _p(y), C, part=stats, split_cp=C if split_out else 0)
        ctx.save_for_backward(x, mean, rstd, gamma, beta, res)
        ctx.cfg = (kind, act, use_batch_stats, ssn)
        ctx.split_out, ctx.grad_split = split_out, grad_split
        if split_out:
            if len(_PRESPLIT_OUT) > 256:
                _PRESPLIT_OUT.clear()
            _PRESPLIT_OUT[y.data_ptr()] = True
        return y

    @staticmethod
    def backward(ctx, gy):
        x, mean, rstd, gamma, beta, res = ctx.saved_tensors
        kind, act, use_stats, ssn = ctx.cfg
        if ctx.split_out:
            gy = gy.contiguous().view(torch.float32)      # fp32 [.., C] gradient that travelled as bf16 [.., 2C]
        gy = as_rows(gy)
        need_gb = gamma is not None and (ctx.needs_input_grad[2] or ctx.needs_input_grad[3])
        gx, dgamma, dbeta, gres = _norm_backward(x, mean, rstd, gamma, beta, res, kind, act, use_stats, ssn, _p(gy), rows_ld(gy)[2],
                                                 ctx.needs_input_grad[0], need_gb, res is not None and ctx.needs_input_grad[7],
                                                 split_cp=x.shape[-1] if ctx.grad_split else 0)
        if ctx.grad_split and gx is not None:
            gx = gx.view(torch.float32)                   # [gx_hi | gx_lo] bf16 data in an fp32 tensor of x's shape
            if not _GY_SPLIT_CB[0]:
                # (entries are consumed by the convolution's backward node a moment later; whatever an interrupted pass leaves
                # behind is dropped when the engine finishes)
                _GY_SPLIT_CB[0] = True
                torch.autograd.Variable._execution_engine.queue_callback(_gy_split_reset)
            _GY_SPLIT_SENT[gx.data_ptr()] = True
        return gx, None, dgamma, dbeta, None, None, None, gres, None, None, None, None, None, None


class NormActCat(torch.autograd.Function):
    """cat((IN(xa) -> act, IN(xb) -> act), channels) in ONE tensor: each half is normalised straight into its channel slice of
    the concatenated output (blocks_MDUNet.conv_3_1, 141-147: the 3^3 and 7^3 branches end in InstanceNorm3d + act and are then
    concatenated for the 1^3 mixer), so no torch.cat copy exists; the backward reads the two slices of the upstream gradient in
    place.  Non-affine instance normalisation only."""

    @staticmethod
    def forward(ctx, xa, xb, act, eps, stats_a=None, stats_b=None):
        _chk_dev(xa, xb)
        xa, xb = as_rows(xa), as_rows(xb)
        ca, cb = xa.shape[-1], xb.shape[-1]
        if xa.shape[:-1] != xb.shape[:-1] or (ca % 8) or (cb % 8):
            raise ValueError("norm_act_cat: operands must share the voxel grid and have channel counts that are multiples of 8")
        y = torch.empty(tuple(xa.shape[:-1]) + (ca + cb,), dtype=xa.dtype, device=xa.device)
        ma, ra, _, ssa = _norm_forward(xa, "instance", None, None, None, None, True, None, act, eps, 0.1, 0, 0, apply=False, part=stats_a)
        mb, rb, _, ssb = _norm_forward(xb, "instance", None, None, None, None, True, None, act, eps, 0.1, 0, 0, apply=False, part=stats_b)
        N = xa.shape[0]
        # one pass over both sources: every 2*(ca+cb)-byte output row is written whole (two launches wrote alternating halves)
        _lib.call("dp_norm_act_cat_fwd", _p(xa), rows_ld(xa)[2], _p(ma), _p(ra), ca, _p(xb), rows_ld(xb)[2], _p(mb), _p(rb), cb, _act_code(act, xa.dtype),
                  _p(y), ca + cb, N, rows_ld(xa)[0] // N, _dt(xa), _stream())
        ctx.save_for_backward(xa, xb, ma, ra, mb, rb)
        ctx.cfg = (act, ssa, ssb)
        return y

    @staticmethod
    def backward(ctx, gy):
        xa, xb, ma, ra, mb, rb = ctx.saved_tensors
        act, ssa, ssb = ctx.cfg
        gy = as_rows(gy)
        ldg, ca = rows_ld(gy)[2], xa.shape[-1]
        ga = gb = None
        if ctx.needs_input_grad[0] and ctx.needs_input_grad[1]:
            # both halves in one pass over whole gradient rows (the per-half passes read 32-byte halves of 64-byte rows)
            cb = xb.shape[-1]
            N = xa.shape[0]
            V = rows_ld(xa)[0] // N
            dev, dtc = xa.device, _dt(xa)
            nblk = _lib.lib().dp_stats_nblk(V)
            part = torch.empty((N, nblk, 2, ca + cb), dtype=torch.float32, device=dev)
            s12 = torch.empty((2, N, ca + cb), dtype=torch.float32, device=dev)
            ga = torch.empty(xa.shape, dtype=xa.dtype, device=dev)
            gb = torch.empty(xb.shape, dtype=xb.dtype, device=dev)
            src = (_p(xa), rows_ld(xa)[2], _p(ma), _p(ra), ca, _p(xb), rows_ld(xb)[2], _p(mb), _p(rb), cb, _p(gy), ldg, _act_code(act, xa.dtype))
            if _lib.call("dp_norm_act_cat_bwd_partial_finalize", *src, N, V, _p(part), _p(s12[0]), _p(s12[1]), dtc, _stream()) == 3:
                _lib.call("dp_norm_act_cat_bwd_partial", *src, N, V, _p(part), dtc, _stream())
                _lib.call("dp_norm_bwd_finalize", _p(part), N, nblk, ca + cb, 0, _p(s12[0]), _p(s12[1]), 0, 0, _stream())
            _lib.call("dp_norm_act_cat_bwd_apply", *src, _p(s12[0]), _p(s12[1]), 1.0 / V, _p(ga), ca, _p(gb), cb, N, V, dtc, _stream())
            return ga, gb, None, None, None, None
        if ctx.needs_input_grad[0]:
            ga = _norm_backward(xa, ma, ra, None, None, None, "instance", act, True, ssa, _p(gy), ldg, True, False, False)[0]
        if ctx.needs_input_grad[1]:
            gb = _norm_backward(xb, mb, rb, None, None, None, "instance", act, True, ssb, gy.data_ptr() + ca * gy.element_size(), ldg,
                                True, False, False)[0]
        return ga, gb, None, None, None, None


def norm_act_cat(xa, xb, act=None, eps=1e-5, stats_a=None, stats_b=None):
    return NormActCat.apply(xa, xb, act, eps, stats_a, stats_b)


def norm_act(x, kind, gamma=None, beta=None, running_mean=None, running_var=None, training=True, res=None, act=None,
             eps=1e-5, momentum=0.1, stats=None, x3_split_for=None):
    """stats: the partial-statistics tensor conv3d(..., stats=True) returned together with x (skips the statistics pass).
    x3_split_for: the nn.Conv3d that is the ONLY consumer of the result.  In the fp32x3 mode, when that convolution takes the x3
    path, the result is written directly as its bf16 [hi | lo] operand (shape [.., 2C]; hand it to conv3d as is) instead of an
    fp32 tensor that the convolution would split in a pass of its own."""
    grad_split = bool(getattr(stats, "_dp_gy_split", False)) and x.dtype == torch.float32
    if kind == "batch" and not training:
        stats = None
    split_out = False
    if x3_split_for is not None and x.dtype == torch.float32 and x.is_cuda:
        from . import config
        c = x3_split_for
        C = x.shape[-1]
        split_out = (config.x3() and C % 16 == 0 and c.weight.shape[1] == C and
                     _x3_conv_shape_ok(x.shape[3], C, c.weight.shape[0], c.kernel_size[0], c.stride[0], c.padding[0], c.dilation[0], _x3_min_w(c.weight)))
    if split_out or grad_split:
        return NormAct.apply(x, kind, gamma, beta, running_mean, running_var, training, res, act, eps, momentum, stats, split_out, grad_split)
    return NormAct.apply(x, kind, gamma, beta, running_mean, running_var, training, res, act, eps, momentum, stats)


class LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        _chk_dev(x)
        x = x.contiguous()
        C = x.shape[-1]
        rows = x.numel() // C
        y = torch.empty_like(x)
        mean = torch.empty((rows,), dtype=torch.float32, device=x.device)
        rstd = torch.empty((rows,), dtype=torch.float32, device=x.device)
        _lib.call("dp_layernorm_fwd", _p(x), _p(gamma.detach()), _p(beta.detach()), _p(y), _p(mean), _p(rstd), rows, C, float(eps),
                  _dt(x), _stream())
        ctx.save_for_backward(x, gamma, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, gamma, mean, rstd = ctx.saved_tensors
        gy = gy.contiguous()
        C = x.shape[-1]
        rows = x.numel() // C
        gx = torch.empty_like(x)
        if _layernorm_det(C):
            dgb = _layernorm_bwd_det(x, gy, None, gamma, mean, rstd, gx, rows, C)
            return gx, dgb[0], dgb[1], None
        dgb = _pass_zeros((2, C), x.device)      # (accumulated by atomics)
        dg, db = dgb[0], dgb[1]
        _lib.call("dp_layernorm_bwd", _p(x), _p(gy), _p(gamma.detach()), _p(mean), _p(rstd), _p(gx), _p(dg), _p(db), rows, C,
                  _dt(x), _stream())
        return gx, dg, db, None


def layer_norm(x, gamma, beta, eps=1e-5):
    return LayerNorm.apply(x, gamma, beta, eps)


def _deterministic():
    from . import config
    return config.deterministic(32)


_LN_DET_MAXC = 1024
_LN_DET_WARNED = [False]


def _layernorm_det(C):
    """True when the LayerNorm backward takes the fixed-order (deterministic) kernel: config.set_deterministic is on AND the row fits it
    (dp_add_layernorm_bwd_det keeps a row in registers: C <= 1024; the reference's hidden size is 768).  Wider rows keep the atomic
    dgamma / dbeta accumulation of dp_layernorm_bwd -- a working model must not turn into an exception because the switch is on
     -- and say so once."""
    if not _deterministic():
        return False
    if C <= _LN_DET_MAXC:
        return True
    if not _LN_DET_WARNED[0]:
        _LN_DET_WARNED[0] = True
        import warnings
        warnings.warn(f"set_deterministic: LayerNorm rows of {C} > {_LN_DET_MAXC} channels accumulate dgamma / dbeta with fp32 atomics "
                      "(run-to-run differences in their last bits); everything else stays deterministic")
    return False


def _layernorm_bwd_det(x, gy, gsum, gamma, mean, rstd, gx, rows, C):
    """config.set_deterministic: LayerNorm backward with dgamma / dbeta through per-block partial rows and a fixed-order combine
    (dp_add_layernorm_bwd_det) instead of fp32 atomics; returns the [2, C] tensor (dgamma, dbeta)."""
    nblk = _lib.lib().dp_layernorm_bwd_parts(rows, C)
    part = torch.empty((nblk, 2, C), dtype=torch.float32, device=x.device)
    dgb = torch.empty((2, C), dtype=torch.float32, device=x.device)
    _lib.call("dp_add_layernorm_bwd_det", _p(x), _p(gy), _p(gsum), _p(gamma.detach()), _p(mean), _p(rstd), _p(gx), _p(part), _p(dgb[0]), _p(dgb[1]),
              rows, C, _dt(x), _stream())
    return dgb


class AddLayerNorm(torch.autograd.Function):
    """(s, z) = (a + b, LayerNorm(a + b)): the residual add of a pre-norm transformer block fused with the LayerNorm that consumes it
    (dp_add_layernorm_fwd / _bwd); the backward adds the residual-path gradient of s inside the LayerNorm backward kernel."""

    @staticmethod
    def forward(ctx, a, b, gamma, beta, eps):
        _chk_dev(a, b)
        ctx.set_materialize_grads(False)      # (an unused output -- the last block's residual sum -- must not cost a zero tensor and a pass over it)
        a, b = a.contiguous(), b.contiguous()
        C = a.shape[-1]
        rows = a.numel() // C
        s, z = torch.empty_like(a), torch.empty_like(a)
        mean = torch.empty((rows,), dtype=torch.float32, device=a.device)
        rstd = torch.empty((rows,), dtype=torch.float32, device=a.device)
        _lib.call("dp_add_layernorm_fwd", _p(a), _p(b), _p(s), _p(gamma.detach()), _p(beta.detach()), _p(z), _p(mean), _p(rstd), rows, C,
                  float(eps), _dt(a), _stream())
        ctx.save_for_backward(s, gamma, mean, rstd)
        return s, z

    @staticmethod
    def backward(ctx, gs, gz):
        s, gamma, mean, rstd = ctx.saved_tensors
        C = s.shape[-1]
        rows = s.numel() // C
        if gz is None:
            return gs, gs, None, None, None           # (also gs is None: nothing flows back)
        gz = gz.contiguous()
        gs = None if gs is None else gs.contiguous()
        gx = torch.empty_like(s)
        if _layernorm_det(C):
            dgb = _layernorm_bwd_det(s, gz, gs, gamma, mean, rstd, gx, rows, C)
            return gx, gx, dgb[0], dgb[1], None
        dgb = _pass_zeros((2, C), s.device)
        if C <= 1024:
            _lib.call("dp_add_layernorm_bwd", _p(s), _p(gz), _p(gs), _p(gamma.detach()), _p(mean), _p(rstd), _p(gx), _p(dgb[0]), _p(dgb[1]),
                      rows, C, _dt(s), _stream())
        else:
            _lib.call("dp_layernorm_bwd", _p(s), _p(gz), _p(gamma.detach()), _p(mean), _p(rstd), _p(gx), _p(dgb[0]), _p(dgb[1]), rows, C,
                      _dt(s), _stream())
            if gs is not None:
                out = torch.empty_like(gx)
                _lib.call("dp_add", _p(gx), _p(gs), _p(out), gx.numel(), gx.numel(), _dt(gx), _stream())
                gx = out
        return gx, gx, dgb[0], dgb[1], None


def add_layer_norm(a, b, gamma, beta, eps=1e-5):
    return AddLayerNorm.apply(a, b, gamma, beta, eps)


# ------------------------------------------------------------------------------------------------ elementwise
class Add(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b):
        a, b = a.contiguous(), b.contiguous()
        y = torch.empty_like(a)
        _lib.call("dp_add", _p(a), _p(b), _p(y), a.numel(), a.numel(), _dt(a), _stream())
        return y

    @staticmethod
    def backward(ctx, g):
        return g, g


def add(a, b):
    return Add.apply(a, b)


class AddBroadcast(torch.autograd.Function):
    """x[B, ...] + p[1, ...] with p an fp32 parameter (position embeddings)."""

    @staticmethod
    def forward(ctx, x, p):
        x = x.contiguous()
        pc = _cast_vec(p.detach().contiguous(), x.dtype)
        y = torch.empty_like(x)
        _lib.call("dp_add", _p(x), _p(pc), _p(y), x.numel(), pc.numel(), _dt(x), _stream())
        ctx.pshape = p.shape
        return y

    @staticmethod
    def backward(ctx, g):
        g = g.contiguous()
        gp = None
        if ctx.needs_input_grad[1]:
            per = 1
            for s in ctx.pshape:
                per *= s
            B = g.numel() // per
            gp = torch.empty(ctx.pshape, dtype=torch.float32, device=g.device)
            _lib.call("dp_sum_batch", _p(g), _p(gp), B, per, _dt(g), _stream())      # fp32 sum over the batch, one pass
        return g, gp


def add_broadcast(x, p):
    return AddBroadcast.apply(x, p)


class Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        x = x.contiguous()
        y = torch.empty_like(x)
        _lib.call("dp_gelu_fwd", _p(x), _p(y), x.numel(), _dt(x), _stream())
        ctx.save_for_backward(x)
        return y

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        g = g.contiguous()
        gx = torch.empty_like(x)
        _lib.call("dp_gelu_bwd", _p(x), _p(g), _p(gx), x.numel(), _dt(x), _stream())
        return gx


def gelu(x):
    return Gelu.apply(x)


# ------------------------------------------------------------------------------------------------ attention
def _transpose(src, lds, sb, dst, ldd, db, rows, cols, nb, dtc):
    _lib.call("dp_transpose", src, lds, sb[0], sb[1], dst, ldd, db[0], db[1], rows, cols, nb[0], nb[1], dtc, _stream())


class Attention(torch.autograd.Function):
    """softmax(q k^T d^-1/2) v of MONAI SABlock on a packed qkv tensor [B, N, 3*H] laid out "(qkv l d)".
    Returns [B, N, H] with heads merged "(l d)".  v1: MFMA GEMMs + row softmax (scores materialised, N <= ~1k)."""

    @staticmethod
    def forward(ctx, qkv, heads):
        _chk_dev(qkv)
        qkv = qkv.contiguous()
        B, N, H3 = qkv.shape
        H = H3 // 3
        d = H // heads
        es = qkv.element_size()
        dtc = _dt(qkv)
        dev = qkv.device
        scale = d ** -0.5
        base = qkv.data_ptr()
        qp, kp, vp = base, base + H * es, base + 2 * H * es
        from . import config as _cfg
        if (_cfg.x3() and _cfg.x3_dgrad_terms() == 1 and qkv.dtype == torch.float32 and d in (64, 128) and not os.environ.get("DP_NO_FUSED_ATTN")
                and not os.environ.get("DP_NO_X3_ATTN_FWD")):
            # fp32x3 (round 5): the fused kernel on the fp32 operands, split into bf16 halves in registers, three products per MFMA step,
            # fp32 output (dp_attention_fwd with DP_X3) -- one launch instead of GEMM + softmax + transpose + GEMM in exact fp32.  The
            # backward pass of this setting (one-product data gradients) needs qkv only.
            O = torch.empty((B, N, H), dtype=torch.float32, device=dev)
            _lib.call("dp_attention_fwd", qp, kp, vp, H3, _p(O), H, 0, B, heads, N, d, float(scale), DP_X3, _stream())
            ctx.fused_bwd = True
            ctx.save_for_backward(qkv)
            ctx.heads = heads
            return O
        S = torch.empty((B, heads, N, N), dtype=qkv.dtype, device=dev)
        bat, sq = (B, heads), (N * H3, d)
        _lib.call("dp_gemm_nt", qp, H3, sq[0], sq[1], kp, H3, sq[0], sq[1], _p(S), N, heads * N * N, N * N, 0, N, N, d, B, heads,
                  1.0, 0, 1, dtc, _stream())
        _lib.call("dp_softmax_fwd", _p(S), _p(S), B * heads * N, N, float(scale), dtc, _stream())
        Vt = torch.empty((B, heads, d, N), dtype=qkv.dtype, device=dev)
        _transpose(vp, H3, sq, _p(Vt), N, (heads * d * N, d * N), N, d, bat, dtc)
        O = torch.empty((B, N, H), dtype=qkv.dtype, device=dev)
        _lib.call("dp_gemm_nt", _p(S), N, heads * N * N, N * N, _p(Vt), N, heads * d * N, d * N, _p(O), H, N * H, d, 0, N, d, N,
                  B, heads, 1.0, 0, 1, dtc, _stream())
        # fp32x3 mode with one-product data gradients (config.set_x3_dgrad_terms, the default): the backward pass runs the fused bf16
        # kernels on the rounded operands -- it needs qkv only (no N x N probabilities kept)
        from . import config as _cfg
        ctx.fused_bwd = bool(_cfg.x3() and _cfg.x3_dgrad_terms() == 1 and qkv.dtype == torch.float32 and d in (64, 128)
                             and not os.environ.get("DP_NO_FUSED_ATTN"))
        if ctx.fused_bwd:
            ctx.save_for_backward(qkv)
        else:
            ctx.save_for_backward(qkv, S)
        ctx.heads = heads
        return O

    @staticmethod
    def backward(ctx, gO):
        heads = ctx.heads
        if ctx.fused_bwd:
            # gy_hi-grade backward: qkv and dO rounded to bf16, the fused forward once more for the log-sum-exp rows and O that belong
            # to THOSE operands (11 us), the fused backward, the result widened to fp32: 5 launches instead of 10 fp32 ones
            (qkv,) = ctx.saved_tensors
            B, N, H3 = qkv.shape
            H = H3 // 3
            d = H // heads
            qh, gOh = _cast_vec(qkv, torch.bfloat16), _cast_vec(gO.contiguous(), torch.bfloat16)
            base = qh.data_ptr()
            Oh = torch.empty((B, N, H), dtype=torch.bfloat16, device=qkv.device)
            lse = torch.empty((B * heads * ((N + 31) // 32 * 32),), dtype=torch.float32, device=qkv.device)
            _lib.call("dp_attention_fwd", base, base + H * 2, base + 2 * H * 2, H3, _p(Oh), H, _p(lse), B, heads, N, d, float(d ** -0.5),
                      _DT[torch.bfloat16], _stream())
            gh = torch.empty_like(qh)
            gb = gh.data_ptr()
            delta = torch.empty_like(lse)
            _lib.call("dp_attention_bwd", base, base + H * 2, base + 2 * H * 2, H3, _p(Oh), _p(gOh), H, _p(lse), _p(delta), gb, gb + H * 2,
                      gb + 2 * H * 2, H3, B, heads, N, d, float(d ** -0.5), _DT[torch.bfloat16], _stream())
            return _cast_vec(gh, torch.float32), None
        qkv, P = ctx.saved_tensors
        gO = gO.contiguous()
        B, N, H3 = qkv.shape
        H = H3 // 3
        d = H // heads
        es = qkv.element_size()
        dtc = _dt(qkv)
        dev = qkv.device
        scale = d ** -0.5
        base = qkv.data_ptr()
        qp, kp, vp = base, base + H * es, base + 2 * H * es
        bat, sq = (B, heads), (N * H3, d)
        sP = (heads * N * N, N * N)
        gqkv = torch.empty_like(qkv)
        gb = gqkv.data_ptr()
        gqp, gkp, gvp = gb, gb + H * es, gb + 2 * H * es
        # dP[q][key] = sum_d dO[q][d] V[key][d]
        dP = torch.empty_like(P)
        _lib.call("dp_gemm_nt", _p(gO), H, N * H, d, vp, H3, sq[0], sq[1], _p(dP), N, sP[0], sP[1], 0, N, N, d, B, heads,
                  1.0, 0, 1, dtc, _stream())
        # dV[key][d] = sum_q P[q][key] dO[q][d]  -> A = P^T [key][q], B = dO^T [d][q]
        Pt = torch.empty_like(P)
        _transpose(_p(P), N, sP, _p(Pt), N, sP, N, N, bat, dtc)
        gOt = torch.empty((B, heads, d, N), dtype=qkv.dtype, device=dev)
        sT = (heads * d * N, d * N)
        _transpose(_p(gO), H, (N * H, d), _p(gOt), N, sT, N, d, bat, dtc)
        _lib.call("dp_gemm_nt", _p(Pt), N, sP[0], sP[1], _p(gOt), N, sT[0], sT[1], gvp, H3, sq[0], sq[1], 0, N, d, N, B, heads,
                  1.0, 0, 1, dtc, _stream())
        # dS = scale * P * (dP - rowsum(dP*P))
        _lib.call("dp_softmax_bwd", _p(P), _p(dP), _p(dP), B * heads * N, N, float(scale), dtc, _stream())
        # dQ[q][d] = sum_key dS[q][key] K[key][d] -> B = K^T [d][key]
        Kt = torch.empty((B, heads, d, N), dtype=qkv.dtype, device=dev)
        _transpose(kp, H3, sq, _p(Kt), N, sT, N, d, bat, dtc)
        _lib.call("dp_gemm_nt", _p(dP), N, sP[0], sP[1], _p(Kt), N, sT[0], sT[1], gqp, H3, sq[0], sq[1], 0, N, d, N, B, heads,
                  1.0, 0, 1, dtc, _stream())
        # dK[key][d] = sum_q dS[q][key] Q[q][d] -> A = dS^T, B = Q^T
        _transpose(_p(dP), N, sP, _p(Pt), N, sP, N, N, bat, dtc)
        Qt = Kt
        _transpose(qp, H3, sq, _p(Qt), N, sT, N, d, bat, dtc)
        _lib.call("dp_gemm_nt", _p(Pt), N, sP[0], sP[1], _p(Qt), N, sT[0], sT[1], gkp, H3, sq[0], sq[1], 0, N, d, N, B, heads,
                  1.0, 0, 1, dtc, _stream())
        return gqkv, None


class FusedAttention(torch.autograd.Function):
    """The same contraction as `Attention` in one launch forward (dp_attention_fwd) and three backward (dp_attention_bwd):
    16-bit storage, head dim 64 or 128; only the per-row log-sum-exp is kept for backward, the N x N scores never exist."""

    @staticmethod
    def forward(ctx, qkv, heads):
        _chk_dev(qkv)
        qkv = qkv.contiguous()
        B, N, H3 = qkv.shape
        H = H3 // 3
        d = H // heads
        es = qkv.element_size()
        base = qkv.data_ptr()
        O = torch.empty((B, N, H), dtype=qkv.dtype, device=qkv.device)
        lse = torch.empty((B * heads * ((N + 31) // 32 * 32),), dtype=torch.float32, device=qkv.device)
        _lib.call("dp_attention_fwd", base, base + H * es, base + 2 * H * es, H3, _p(O), H, _p(lse), B, heads, N, d, float(d ** -0.5),
                  _dt(qkv), _stream())
        ctx.save_for_backward(qkv, O, lse)
        ctx.heads = heads
        return O

    @staticmethod
    def backward(ctx, gO):
        qkv, O, lse = ctx.saved_tensors
        heads = ctx.heads
        gO = gO.contiguous()
        B, N, H3 = qkv.shape
        H = H3 // 3
        d = H // heads
        es = qkv.element_size()
        base = qkv.data_ptr()
        gqkv = torch.empty_like(qkv)
        gb = gqkv.data_ptr()
        delta = torch.empty_like(lse)
        _lib.call("dp_attention_bwd", base, base + H * es, base + 2 * H * es, H3, _p(O), _p(gO), H, _p(lse), _p(delta), gb, gb + H * es,
                  gb + 2 * H * es, H3, B, heads, N, d, float(d ** -0.5), _dt(qkv), _stream())
        return gqkv, None


def attention(qkv, heads):
    """MONAI SABlock core on the packed qkv Linear output.  16-bit storage with head dim 64 / 128 (every configuration of
    BASELINE.json) takes the fused kernels; fp32 (parity mode) and other head dims take MFMA GEMMs + row softmax."""
    d = qkv.shape[-1] // 3 // heads
    if qkv.dtype != torch.float32 and d in (64, 128) and not os.environ.get("DP_NO_FUSED_ATTN"):
        return FusedAttention.apply(qkv, heads)
    return Attention.apply(qkv, heads)


# ------------------------------------------------------------------------------------------------ rotary positions, norm of queries and keys
_POS_KIND = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
HEAD_DIMS = (32, 64, 96, 128)


def _device_of(t):
    """Context in which launches go to t's device (nothing to do where it is the current one)."""
    if _raw_device is not None and t.get_device() == _raw_device():
        return _NO_GUARD
    return torch.cuda.device(t.device)


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


_NO_GUARD = _NoGuard()


class _NoContext:
    """What forward() writes into where no backward pass can follow."""
    needs_input_grad = (False,) * 16

    def save_for_backward(self, *tensors):
        return None


def _run(fn, leaves, *args):
    """fn.apply(*leaves, *args), without a node of the graph where none of the leaves asks for a gradient (a call: 11.9 us of host time instead of 15.6).
    A recording (torch.jit.trace) holds the node or nothing of the call, and forward-mode derivatives are refused by it: both always get it (also where
    torch does not say whether a forward-mode level is open)."""
    if getattr(_fwd_ad, "_current_level", 0) < 0 and not torch.jit.is_tracing():
        if not torch.is_grad_enabled():
            return fn.forward(_NoContext(), *leaves, *args)
        for t in leaves:
            if t is not None and t.requires_grad:
                break
        else:
            return fn.forward(_NoContext(), *leaves, *args)
    return fn.apply(*leaves, *args)


class _NoSecondDerivative(torch.autograd.Function):
    """Gradients that were asked for with a graph: the same tensors, behind a node that refuses to be passed."""

    @staticmethod
    def forward(ctx, what, leaf, *grads):
        ctx.what = what
        return grads

    @staticmethod
    def backward(ctx, *gs):
        raise RuntimeError(f"{ctx.what}: the second derivative is not defined (its gradients are constants to autograd)")


def _first_order(backward):
    """backward() of an operator whose gradients cannot be differentiated again: with create_graph=True they say so when it is tried."""
    @functools.wraps(backward)
    def wrapper(ctx, *gs):
        if not torch.is_grad_enabled():
            return backward(ctx, *gs)
        with torch.no_grad():
            grads = backward(ctx, *gs)
        behind = iter(_NoSecondDerivative.apply(backward.__qualname__.split(".")[0], torch.empty(0, requires_grad=True), *(g for g in grads if g is not None)))
        return tuple(None if g is None else next(behind) for g in grads)
    return wrapper


def _strided(t, tiles=False):
    """(tensor, strides of all but the last dimension): t itself where its last dimension is dense and every row 16-byte aligned (tiles: and
    its tokens, dimension 1, do not overlap and lie at most 16 MB apart), otherwise a contiguous copy."""
    st, es, shape = t.stride(), t.element_size(), t.shape
    if t.data_ptr() % 16 == 0 and (st[-1] == 1 or shape[-1] <= 1):
        if 1 not in shape[:-1] and t.is_contiguous() and st[-2] * es % 16 == 0 and t.numel():
            return t, st[:-1]      # (the stride of a dimension of one may be anything, in a contiguous tensor too: below)
        if all(n <= 1 or s * es % 16 == 0 for n, s in zip(shape[:-1], st)) and not (
                tiles and shape[1] > 1 and (st[1] < shape[-1] or st[1] * es > 1 << 24)):
            return t, [0 if n <= 1 else s for n, s in zip(shape[:-1], st)]
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()[:-1]


# (The functions check their arguments in forward(): a recorded call comes in there again, with tensors of other sizes.  Sizes are made ints there,
# because they are tensors while a recording runs.)
def _head_dim(width, heads, what):
    if heads < 1 or width % heads:
        raise ValueError(f"{what}: {width} channels do not divide into {heads} heads")
    d = width // heads
    if d not in HEAD_DIMS:
        raise ValueError(f"{what}: head dim {d} not in {HEAD_DIMS}")
    return d


@functools.lru_cache(maxsize=256)
def _rotary_plan(what, d, sections, base, interleaved):
    """The part of the C ABI's arguments that depends on the configuration alone (checked once per configuration)."""
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or 2 * sum(sections) > d:
        raise ValueError(f"{what}: sections {sections} of a head of {d} channels (1 to 4 axes, at most {d // 2} pairs)")
    if not 1.0 < float(base) < 1e30:
        raise ValueError(f"{what}: base {base}")
    return (len(sections), *(int(n) for n in sections), *(0,) * (4 - len(sections)), float(base), int(bool(interleaved)))


_NO_ROTARY = (0, 0, 0, 0, 0, 0, 0, 0.0, 0)


def _rotary_args(what, x, d, positions, sections, base, interleaved):
    """(positions tensor, the C ABI's arguments behind the pointer) of a rotation; (None, ...) without one."""
    if positions is None:
        if sections is not None:
            raise ValueError(f"{what}: sections without positions")
        return None, _NO_ROTARY
    if sections is None:
        raise ValueError(f"{what}: positions need sections (rotated pairs of a head per axis)")
    plan = _rotary_plan(what, d, tuple(sections), base, interleaved)
    (B, N), shape, axes = map(int, x.shape[:2]), tuple(map(int, positions.shape)), plan[0]
    kind = _POS_KIND.get(positions.dtype)
    if kind is None:
        raise TypeError(f"{what}: positions are int32, int64 or float32, got {positions.dtype}")
    if positions.device != x.device:
        raise _lib.DoseHipError(f"{what}: positions on {positions.device}, rows on {x.device}")
    if len(shape) not in (2, 3) or shape[-2] != N or shape[-1] != axes or (len(shape) == 3 and shape[0] not in (1, B)):
        raise ValueError(f"{what}: positions {tuple(shape)} for {B} x {N} tokens and {axes} axes")
    return positions.contiguous(), (kind, N * axes if len(shape) == 3 and shape[0] == B else 0, *plan)


def _check_norm(what, x, d, *ws):
    for w in ws:
        if w is None:
            raise ValueError(f"{what}: the norm has a weight and a bias for queries and for keys, one of them is None")
        if w.dtype != torch.float32 or w.dim() != 1 or w.shape[0] != d:
            raise ValueError(f"{what}: the norm's weights and biases are float32 [{d}], got {w.dtype} {tuple(w.shape)}")
        if w.device != x.device:
            raise _lib.DoseHipError(f"{what}: the norm's weights on {w.device}, rows on {x.device}")


def _dense(*ws):
    """Weights as the kernels read them: dense, 16-byte aligned (themselves, as a rule)."""
    return [w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.detach().clone(memory_format=torch.contiguous_format) for w in ws]


class RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, heads, positions, sections, base, interleaved):
        what = "rotary_axes"
        _dt(x)
        if x.dim() != 3:
            raise ValueError(f"{what}: x is [B, N, channels], got {tuple(x.shape)}")
        B, N, W = map(int, x.shape)
        d = _head_dim(W, heads, what)
        positions, rot = _rotary_args(what, x, d, positions, sections, base, interleaved)
        _chk_dev(x)
        xs, (xb, xt) = _strided(x)
        y = x.new_empty((B, N, W))
        with _device_of(x):
            _lib.call("dp_qk_rotary_fwd", _p(xs), xb, xt, _p(y), N * W, W, B, N, heads, 0, d, 0, 0, 0, 0, 0.0, _p(positions), *rot, 0,
                      _dt(x), _stream())
        ctx.save_for_backward(positions)
        ctx.heads, ctx.rot = heads, rot
        return y

    @staticmethod
    @_first_order
    def backward(ctx, g):
        (positions,) = ctx.saved_tensors
        gs, (gb, gt) = _strided(g)
        B, N, W = g.shape
        gx = g.new_empty((B, N, W))
        with _device_of(g):
            _lib.call("dp_qk_rotary_fwd", _p(gs), gb, gt, _p(gx), N * W, W, B, N, ctx.heads, 0, W // ctx.heads, 0, 0, 0, 0, 0.0, _p(positions),
                      *ctx.rot, 1, _dt(g), _stream())
        return gx, None, None, None, None, None


def rotary_axes(x, heads, positions, sections, base=10000.0, interleaved=False):
    """Rotary positions over the axes of a token grid: x [B, N, heads * d] (rows may be slices of wider ones) with every pair of a head turned
    by its token's angle.  positions [N, axes] or [B, N, axes] (int32, int64 or float32); sections: rotated pairs of a head per axis -- pair e
    of an axis with n pairs turns by position * base^(-e / n); pairs behind the sections stay.  interleaved False: pair i = channels
    (i, i + d / 2), True: (2 i, 2 i + 1).  d in HEAD_DIMS.  The gradient is the turn backwards; positions have none."""
    return _run(RotaryAxes, (x,), int(heads), positions, sections, base, interleaved)


class QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, qw, qb, kw, kb, heads, kv, eps, positions, sections, base, interleaved):
        what = "qk_norm_rotary"
        _dt(x)
        if x.dim() != 3 or heads < 1 or kv < 1:
            raise ValueError(f"{what}: x is [B, N, channels] with heads and kv_heads of at least 1, got {tuple(x.shape)}, {heads}, {kv}")
        B, N, W = map(int, x.shape)
        d = _head_dim(W, heads + kv, what)
        _check_norm(what, x, d, qw, qb, kw, kb)
        positions, rot = _rotary_args(what, x, d, positions, sections, base, interleaved)
        _chk_dev(x, qw, qb, kw, kb)
        xs, (xb, xt) = _strided(x)
        qwd, qbd, kwd, kbd = _dense(qw, qb, kw, kb)
        y = x.new_empty((B, N, W))
        with _device_of(x):
            _lib.call("dp_qk_rotary_fwd", _p(xs), xb, xt, _p(y), N * W, W, B, N, heads, kv, d, _p(qwd), _p(qbd), _p(kwd), _p(kbd), eps,
                      _p(positions), *rot, 0, _dt(x), _stream())
        ctx.save_for_backward(xs, qw, kw, positions)
        ctx.opts = (xb, xt, heads, kv, eps, rot)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, g):
        xs, qw, kw, positions = ctx.saved_tensors
        xb, xt, heads, kv, eps, rot = ctx.opts
        gs, (gb, gt) = _strided(g)
        B, N, W = g.shape
        d = W // (heads + kv)
        qwd, kwd = _dense(qw, kw)
        gx = g.new_empty((B, N, W))
        dw = g.new_empty((4, d), dtype=torch.float32)
        part = g.new_empty((_lib.lib().dp_qk_rotary_parts(B * N), 4, d), dtype=torch.float32)
        with _device_of(g):
            _lib.call("dp_qk_rotary_bwd", _p(xs), xb, xt, _p(gs), gb, gt, 0, _p(gx), N * W, W, _p(part), _p(dw), B, N, heads, kv, d, _p(qwd),
                      _p(kwd), eps, _p(positions), *rot, _dt(g), _stream())
        return (gx, *dw.unbind(0), None, None, None, None, None, None, None)


def qk_norm_rotary(x, heads, kv_heads, q_weight, q_bias, k_weight, k_bias, eps=1e-5, positions=None, sections=None, base=10000.0,
                   interleaved=False):
    """LayerNorm of every head of queries and keys -- x [B, N, (heads + kv_heads) * d], rows may be slices of wider ones; one float32 [d]
    weight and bias for all query heads, one for all key heads -- and, with positions, the rotation of rotary_axes behind it, in one pass.
    The weights' gradients are added up in a fixed order."""
    return _run(QkNormRotary, (x, q_weight, q_bias, k_weight, k_bias), int(heads), int(kv_heads), float(eps), positions, sections, base, interleaved)


# ------------------------------------------------------------------------------------------------ attention over a sliding window
def _per_sequence(what, name, t, B, like):
    """int32 [B] on the rows' device."""
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64) or tuple(t.shape) != (B,):
        raise ValueError(f"{what}: {name} is int32 or int64 [{B}], got {t.dtype} {tuple(t.shape)}")
    if t.device != like.device:
        raise _lib.DoseHipError(f"{what}: {name} on {t.device}, rows on {like.device}")
    if t.dtype == torch.int64:
        t = t.clamp(-(1 << 30), 1 << 30)      # (a number past 32 bits stays past every row)
    return t.to(torch.int32).contiguous()


def _window_args(what, left, right, sinks, scale, d):
    for name, v in (("left", left), ("right", right)):
        if v is not None and not 0 <= int(v) < 1 << 31:
            raise ValueError(f"{what}: {name} is None or at least 0, got {v}")
    left, right = (-1 if v is None else int(v) for v in (left, right))
    sinks = int(sinks)
    if not 0 <= sinks < 1 << 31:
        raise ValueError(f"{what}: sinks {sinks}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"{what}: scale {scale}")
    return left, right, sinks, scale


def _window_ws(B, heads, kv, Nq, Nk, d, win, backward, dev):
    n = _lib.lib().dp_window_attention_ws_elems(B, heads, kv, Nq, Nk, d, win[0], win[1], win[2], backward)
    return torch.empty((n,), dtype=torch.float32, device=dev) if n else None


class WindowAttention(torch.autograd.Function):
    """q [B, Nq, heads, d], k / v [B, Nk, kv, d]."""

    @staticmethod
    def forward(ctx, q, k, v, left, right, sinks, scale, start, lengths):
        what = "window_attention"
        _dt(q)
        if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
            raise ValueError(f"{what}: q [B, Nq, heads, d], k and v [B, Nk, kv_heads, d], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
        if not q.dtype == k.dtype == v.dtype or not q.device == k.device == v.device:
            raise TypeError(f"{what}: q, k and v share type and device, got {q.dtype}, {k.dtype}, {v.dtype} on {q.device}, {k.device}, {v.device}")
        (B, Nq, heads, d), (Nk, kv) = map(int, q.shape), map(int, k.shape[1:3])
        if heads < 1 or kv < 1 or heads % kv:
            raise ValueError(f"{what}: {heads} query heads do not divide over {kv} key heads")
        _head_dim(heads * d, heads, what)
        win = _window_args(what, left, right, sinks, scale, d)
        starts = None
        if torch.is_tensor(start):
            starts, start = _per_sequence(what, "q_start", start, B, q), 0
        start = int(start)
        if abs(start) >= 1 << 30:
            raise ValueError(f"{what}: q_start {start}")
        lengths = _per_sequence(what, "lengths", lengths, B, q)
        _chk_dev(q)
        (qs, qst), (ks, kst), (vs, vst) = _strided(q, True), _strided(k, True), _strided(v, True)
        o = q.new_empty((B, Nq, heads, d))
        need = any(ctx.needs_input_grad[:3])
        lse = q.new_empty((B * heads * Nq,), dtype=torch.float32) if need else None
        with _device_of(q):
            ws = _window_ws(B, heads, kv, Nq, Nk, d, win, 0, q.device)
            _lib.call("dp_window_attention_fwd", _p(qs), *qst, _p(ks), *kst, _p(vs), *vst, _p(o), Nq * heads * d, heads * d, d, _p(lse), _p(ws),
                      B, heads, kv, Nq, Nk, d, win[0], win[1], win[2], start, _p(starts), _p(lengths), win[3], _dt(q), _stream())
        if need:
            ctx.save_for_backward(qs, ks, vs, o, lse, starts, lengths)
            ctx.opts = (qst, kst, vst, win, start)
        return o

    @staticmethod
    @_first_order
    def backward(ctx, g):
        q, k, v, o, lse, starts, lengths = ctx.saved_tensors
        qst, kst, vst, win, start = ctx.opts
        gs, gst = _strided(g, True)
        (B, Nq, heads, d), (Nk, kv) = q.shape, k.shape[1:3]
        dq = q.new_empty((B, Nq, heads, d))
        dk = q.new_empty((B, Nk, kv, d))
        dv = torch.empty_like(dk)
        delta = torch.empty_like(lse)
        with _device_of(q):
            ws = _window_ws(B, heads, kv, Nq, Nk, d, win, 1, q.device)
            _lib.call("dp_window_attention_bwd", _p(q), *qst, _p(k), *kst, _p(v), *vst, _p(o), Nq * heads * d, heads * d, d, _p(gs), *gst, _p(lse),
                      _p(delta), _p(dq), Nq * heads * d, heads * d, d, _p(dk), Nk * kv * d, kv * d, d, _p(dv), Nk * kv * d, kv * d, d, 0, _p(ws), B,
                      heads, kv, Nq, Nk, d, win[0], win[1], win[2], start, _p(starts), _p(lengths), win[3], _dt(q), _stream())
        return dq, dk, dv, None, None, None, None, None, None


def window_attention(q, k, v, left=None, right=None, sinks=0, q_start=0, lengths=None, scale=None):
    """softmax(scale q k^T) v over a sliding window, whose first tokens stay visible.  q [B, Nq, heads, d], k and v [B, Nk, kv_heads, d] (any
    strides; heads % kv_heads == 0: that many query heads share a key head; d in HEAD_DIMS); returns [B, Nq, heads, d].

    The query in row i stands at position p = q_start + i (q_start: an int, or int32 / int64 [B]) and sees key j iff j < lengths[b],
    j <= p + right, and j >= p - left or j < sinks.  left / right None: no limit on that side; right=0 looks back only.  lengths (int32 /
    int64 [B], None: all Nk keys): rows at positions outside [0, lengths[b]) give 0 and get and cause no gradient, whatever they hold, NaN
    included.  (A value that is not finite inside a sequence reaches the rows it is seen by, and may reach others near them.)
    scale None: d^-1/2.  Sums are added in a fixed order: the same inputs give the same bits."""
    return _run(WindowAttention, (q, k, v), left, right, sinks, scale, q_start, lengths)


def check_attention_options(width, heads, left, right, sinks, sections, base, interleaved):
    """What window_attention_qkv checks of a configuration, for a module to check when it is built."""
    what = "window_attention_qkv"
    d = _head_dim(width, heads, what)
    _window_args(what, left, right, sinks, None, d)
    if sections is not None:
        _rotary_plan(what, d, tuple(sections), base, interleaved)


class WindowAttentionQkv(torch.autograd.Function):
    """The packed projection's form: norm and rotation of q and k into a buffer of their own (one launch, none without them), v read in
    place; the backward pass writes one packed gradient, that of q and k passing through the norm and the rotation unrounded (float).
    The buffer holds q and k in the storage type, which is what the matrix cores take: in 16 bits half a step of each behind the turn
    (bf16, 4097 tokens: the result is off by 3.6e-3 in the 2-norm, by 2.4e-3 where q and k come rounded anyway)."""

    @staticmethod
    def forward(ctx, qkv, qw, qb, kw, kb, heads, kv, eps, positions, sections, base, interleaved, left, right, sinks, scale, lengths):
        what, es, dtc = "window_attention_qkv", qkv.element_size(), _dt(qkv)
        if qkv.dim() != 3 or heads < 1 or kv < 1 or heads % kv:
            raise ValueError(f"{what}: qkv is [B, N, channels] and kv_heads divides heads, got {tuple(qkv.shape)}, {heads}, {kv}")
        B, N, W = map(int, qkv.shape)
        d = _head_dim(W, heads + 2 * kv, what)
        if any(w is not None for w in (qw, qb, kw, kb)):
            _check_norm(what, qkv, d, qw, qb, kw, kb)
        positions, rot = _rotary_args(what, qkv, d, positions, sections, base, interleaved)
        win = _window_args(what, left, right, sinks, scale, d)
        lengths = _per_sequence(what, "lengths", lengths, B, qkv)
        _chk_dev(qkv, qw, qb, kw, kb)
        xs, (xb, xt) = _strided(qkv, True)
        Wq, Wqk = heads * d, (heads + kv) * d
        pre = qw is not None or positions is not None
        o = qkv.new_empty((B, N, Wq))
        need = any(ctx.needs_input_grad[:5])
        lse = qkv.new_empty((B * heads * N,), dtype=torch.float32) if need else None
        with _device_of(qkv):
            qk, qkb, qkt = xs, xb, xt
            if pre:
                ws4 = _dense(qw, qb, kw, kb) if qw is not None else (None,) * 4
                qk, qkb, qkt = qkv.new_empty((B, N, Wqk)), N * Wqk, Wqk
                _lib.call("dp_qk_rotary_fwd", _p(xs), xb, xt, _p(qk), qkb, qkt, B, N, heads, kv, d, *(_p(w) for w in ws4), eps, _p(positions), *rot,
                          0, dtc, _stream())
            ws = _window_ws(B, heads, kv, N, N, d, win, 0, qkv.device)
            _lib.call("dp_window_attention_fwd", _p(qk), qkb, qkt, d, _p(qk) + Wq * es, qkb, qkt, d, _p(xs) + Wqk * es, xb, xt, d, _p(o), N * Wq, Wq, d,
                      _p(lse), _p(ws), B, heads, kv, N, N, d, win[0], win[1], win[2], 0, 0, _p(lengths), win[3], dtc, _stream())
        if need:
            ctx.save_for_backward(xs, qk if pre else None, o, lse, qw, kw, positions, lengths)
            ctx.opts = (xb, xt, heads, kv, eps, rot, win)
        return o

    @staticmethod
    @_first_order
    def backward(ctx, g):
        xs, qk, o, lse, qw, kw, positions, lengths = ctx.saved_tensors
        xb, xt, heads, kv, eps, rot, win = ctx.opts
        gs, (gb, gt) = _strided(g, True)
        B, N, W = xs.shape
        d, es, dtc = W // (heads + 2 * kv), xs.element_size(), _dt(xs)
        Wq, Wqk = heads * d, (heads + kv) * d
        gx = xs.new_empty((B, N, W))
        delta = torch.empty_like(lse)
        dw = None
        with _device_of(xs):
            ws = _window_ws(B, heads, kv, N, N, d, win, 1, xs.device)
            src, sb, stt = (xs, xb, xt) if qk is None else (qk, N * Wqk, Wqk)
            # dq, dk: into the packed gradient, or (16-bit storage, norm / rotation still to come) into a float buffer
            wide = qk is not None and xs.dtype != torch.float32
            dst, db, dt_, des = (xs.new_empty((B, N, Wqk), dtype=torch.float32), N * Wqk, Wqk, 4) if wide else (gx, N * W, W, es)
            _lib.call("dp_window_attention_bwd", _p(src), sb, stt, d, _p(src) + Wq * es, sb, stt, d, _p(xs) + Wqk * es, xb, xt, d, _p(o), N * Wq, Wq, d,
                      _p(gs), gb, gt, d, _p(lse), _p(delta), _p(dst), db, dt_, d, _p(dst) + Wq * des, db, dt_, d, _p(gx) + Wqk * es, N * W, W, d,
                      1 if wide else 0, _p(ws), B, heads, kv, N, N, d, win[0], win[1], win[2], 0, 0, _p(lengths), win[3], dtc, _stream())
            if qk is not None:
                part = None
                if qw is not None:
                    qw, kw = _dense(qw, kw)
                    dw = xs.new_empty((4, d), dtype=torch.float32)
                    part = xs.new_empty((_lib.lib().dp_qk_rotary_parts(B * N), 4, d), dtype=torch.float32)
                _lib.call("dp_qk_rotary_bwd_ragged", _p(xs), xb, xt, _p(dst), db, dt_, 1 if wide else 0, _p(gx), N * W, W, _p(part), _p(dw), B, N, heads,
                          kv, d, _p(qw), _p(kw), eps, _p(positions), *rot, _p(lengths), dtc, _stream())
        return (gx, *(dw.unbind(0) if dw is not None else (None,) * 4), *(None,) * 12)


def window_attention_qkv(qkv, heads, kv_heads=None, left=None, right=None, sinks=0, lengths=None, scale=None, norm=None, eps=1e-5,
                         positions=None, sections=None, base=10000.0, interleaved=False):
    """The attention block's core on the packed projection [B, N, (heads + 2 kv_heads) * d] ("q heads | k heads | v heads", kv_heads None:
    as many as heads), as attention() takes it: with norm = (q_weight, q_bias, k_weight, k_bias) the LayerNorm of qk_norm_rotary, with
    positions the rotation of rotary_axes, then window_attention of the rows with themselves.  Returns [B, N, heads * d].  Rows outside
    [0, lengths[b]) add nothing to the norm's gradients either, whatever they and their positions hold."""
    what = "window_attention_qkv"
    norm = tuple(norm) if norm is not None else (None,) * 4
    if len(norm) != 4:
        raise ValueError(f"{what}: norm is (q_weight, q_bias, k_weight, k_bias)")
    return _run(WindowAttentionQkv, (qkv, *norm), int(heads), int(heads if kv_heads is None else kv_heads), float(eps), positions, sections, base,
                interleaved, left, right, sinks, scale, lengths)


# ------------------------------------------------------------------------------------------------ misc
class Patchify(torch.autograd.Function):
    """einops "b c (h p1)(w p2)(d p3) -> b (h w d)(p1 p2 p3 c)" on an NDHWC tensor (first C channels)."""

    @staticmethod
    def forward(ctx, x, C, p):
        x = as_rows(x)
        _, cx, ld = rows_ld(x)
        B, S0, S1, S2 = x.shape[:4]
        ntok = (S0 // p) * (S1 // p) * (S2 // p)
        out = torch.empty((B, ntok, p * p * p * C), dtype=x.dtype, device=x.device)
        _lib.call("dp_patchify", _p(x), _p(out), B, S0, S1, S2, C, ld, p, _dt(x), _stream())
        ctx.cfg = (tuple(x.shape), C, p)
        return out

    @staticmethod
    def backward(ctx, g):
        shape, C, p = ctx.cfg
        g = g.contiguous()
        gx = torch.zeros(shape, dtype=g.dtype, device=g.device) if shape[-1] > C else torch.empty(shape, dtype=g.dtype, device=g.device)
        _lib.call("dp_unpatchify", _p(g), _p(gx), shape[0], shape[1], shape[2], shape[3], C, shape[-1], p, _dt(g), _stream())
        return gx, None, None


def patchify(x, C, p=16):
    return Patchify.apply(x, C, p)


class TrilinearUp2(torch.autograd.Function):
    """F.interpolate(scale_factor=2, mode='trilinear', align_corners=True) (c3d.py:36)."""

    @staticmethod
    def forward(ctx, x):
        x = as_rows(x)
        _, C, ld = rows_ld(x)
        N, D, H, W = x.shape[:4]
        y = torch.empty((N, 2 * D, 2 * H, 2 * W, C), dtype=x.dtype, device=x.device)
        _lib.call("dp_trilinear_up2_fwd", _p(x), ld, _p(y), C, N, D, H, W, C, _dt(x), _stream())
        ctx.shape = tuple(x.shape)
        return y

    @staticmethod
    def backward(ctx, g):
        g = as_rows(g)
        _, C, ldg = rows_ld(g)
        N, D, H, W, _ = ctx.shape
        acc = torch.zeros(ctx.shape, dtype=torch.float32, device=g.device)
        _lib.call("dp_trilinear_up2_bwd", _p(g), ldg, _p(acc), N, D, H, W, C, _dt(g), _stream())
        if g.dtype == torch.float32:
            return acc
        gx = torch.empty(ctx.shape, dtype=g.dtype, device=g.device)
        _lib.call("dp_cast", _p(acc), 0, _p(gx), _dt(g), acc.numel(), _stream())
        return gx


def trilinear_up2(x, x3_split_for=None):
    """x3_split_for: the nn.Conv3d that is the ONLY consumer of the result.  In the fp32x3 mode, when no gradient flows through (the frozen C3D of
    DOSE-PYFER, train_light_pyfer.py:85-88; inference) and that convolution takes the x3 path, the result is written directly as its bf16
    [hi | lo] operand (shape [.., 2 C]; hand it to conv3d as is): the fp32 up-sampled tensor -- 1.07 GB at 2 x 128^3 x 32 channels -- and the
    split pass over it do not exist (round 6: 0.25 ms of the fp32x3 step at the 128^3 level alone)."""
    if x3_split_for is not None and x.dtype == torch.float32 and x.is_cuda and not (torch.is_grad_enabled() and x.requires_grad):
        from . import config
        c = x3_split_for
        C = x.shape[-1]
        if (config.x3() and C % 16 == 0 and c.weight.shape[1] == C and not (torch.is_grad_enabled() and c.weight.requires_grad) and
                _x3_conv_shape_ok(2 * x.shape[3], C, c.weight.shape[0], c.kernel_size[0], c.stride[0], c.padding[0], c.dilation[0], _x3_min_w(c.weight))):
            x = as_rows(x)
            _, _, ld = rows_ld(x)
            N, D, H, W = x.shape[:4]
            y = torch.empty((N, 2 * D, 2 * H, 2 * W, 2 * C), dtype=torch.bfloat16, device=x.device)
            _lib.call("dp_trilinear_up2_fwd", _p(x), ld, _p(y), 2 * C, N, D, H, W, C, DP_X3, _stream())
            if len(_PRESPLIT_OUT) > 256:
                _PRESPLIT_OUT.clear()
            _PRESPLIT_OUT[y.data_ptr()] = True
            return y
    return TrilinearUp2.apply(x)


def argmax_onehot(logits, out=None, choff=0, labels=False):
    """Cascade glue (train_light_linked_model.py:157-167): arg-max over channels -> one-hot of classes 1..C-1 written
    into channels [choff, choff+C-1) of ``out`` (NDHWC); optionally also the int32 label volume."""
    logits = as_rows(logits)
    rows, C, ld = rows_ld(logits)
    lab = torch.empty(tuple(logits.shape[:-1]), dtype=torch.int32, device=logits.device) if labels else None
    ldo = 0
    if out is not None:
        ldo = rows_ld(out)[2]
    if out is not None and out.dtype != logits.dtype:
        _lib.call("dp_argmax_onehot2", _p(logits), ld, _dt(logits), _p(out), ldo, _dt(out), choff, _p(lab), rows, C, _stream())
    else:
        _lib.call("dp_argmax_onehot", _p(logits), ld, _p(out), ldo, choff, _p(lab), rows, C, _dt(logits), _stream())
    return lab


# ------------------------------------------------------------------------------------------------ loss / metrics
class MaskedL1(torch.autograd.Function):
    """mean |pred - gt| over mask > 0 (Train/loss.py:13-28, 69-107) without boolean indexing: dp_masked_l1_fwd / _bwd; with
    huber_delta > 0 the element is nn.HuberLoss(delta)'s (loss.py:53: GenLoss(huber=True)), dp_masked_huber_fwd / _bwd.
    pred, gt, mask: fp32 device tensors of equal numel (any shape); returns a 0-dim fp32 tensor."""

    @staticmethod
    def forward(ctx, pred, gt, mask, huber_delta):
        _chk_dev(pred, gt, mask)
        if pred.dtype != torch.float32:
            raise _lib.DoseHipError("masked_l1 takes the fp32 tensors of the module boundary")
        pred, gt, mask = pred.contiguous(), gt.contiguous().float(), mask.contiguous().float()
        n = pred.numel()
        if gt.numel() != n or mask.numel() != n:
            raise ValueError("masked_l1: pred, gt and mask must have the same number of elements")
        ws = torch.empty((_lib.lib().dp_masked_l1_ws_elems(n),), dtype=torch.float32, device=pred.device)
        out = torch.empty((3,), dtype=torch.float32, device=pred.device)
        if huber_delta > 0:
            _lib.call("dp_masked_huber_fwd", _p(pred), _p(gt), _p(mask), n, float(huber_delta), _p(ws), _p(out), _stream())
        else:
            _lib.call("dp_masked_l1_fwd", _p(pred), _p(gt), _p(mask), n, _p(ws), _p(out), 0, _stream())
        ctx.save_for_backward(pred, gt, mask, out)
        ctx.delta = float(huber_delta)
        return out[2]

    @staticmethod
    def backward(ctx, g):
        pred, gt, mask, out = ctx.saved_tensors
        gp = torch.empty_like(pred)
        gup = g.contiguous().float().reshape(1)
        if ctx.delta > 0:
            _lib.call("dp_masked_huber_bwd", _p(pred), _p(gt), _p(mask), _p(out), _p(gup), _p(gp), pred.numel(), ctx.delta, _stream())
        else:
            _lib.call("dp_masked_l1_bwd", _p(pred), _p(gt), _p(mask), _p(out), _p(gup), _p(gp), pred.numel(), _stream())
        return gp, None, None, None


def masked_l1(pred, gt, mask, huber_delta=0.0):
    return MaskedL1.apply(pred, gt, mask, huber_delta)


_LABEL_KIND = {torch.float32: 0, torch.int64: 1, torch.int32: 2, torch.uint8: 3}


class DiceCE(torch.autograd.Function):
    """monai.losses.DiceCELoss(to_onehot_y=True, softmax=True) (OARSegmentation/train_light_transeg.py:148,196): one fused pass over the
    logits forward (softmax, cross-entropy term, the three Dice sums per class) and one backward (dp_dice_ce_fwd / _bwd).
    logits: fp32 [B, C, D, H, W] (the module boundary's NCDHW tensor); labels: [B, 1, D, H, W] or [B, D, H, W] class indices stored
    as float32 (the reference's loader), int64, int32 or uint8.  Returns the 0-dim fp32 loss."""

    @staticmethod
    def forward(ctx, logits, labels, smooth_nr, smooth_dr, lambda_dice, lambda_ce):
        _chk_dev(logits, labels)
        if logits.dtype != torch.float32:
            raise _lib.DoseHipError("dice_ce takes the fp32 logits of the module boundary")
        logits = logits.contiguous()
        B, C = logits.shape[:2]
        V = logits.numel() // (B * C)
        if labels.dtype not in _LABEL_KIND:
            labels = labels.to(torch.int32)
        labels = labels.contiguous()
        if labels.numel() != B * V:
            raise ValueError("dice_ce: labels must hold one class index per voxel ([B, 1, ...] or [B, ...])")
        L = _lib.lib()
        ws = torch.empty((L.dp_dice_ce_ws_elems(B, C, V),), dtype=torch.float32, device=logits.device)
        stats = torch.empty((L.dp_dice_ce_stats_elems(B, C),), dtype=torch.float32, device=logits.device)
        _lib.call("dp_dice_ce_fwd", _p(logits), _p(labels), _LABEL_KIND[labels.dtype], B, C, V, float(smooth_nr), float(smooth_dr),
                  float(lambda_dice), float(lambda_ce), _p(ws), _p(stats), _stream())
        ctx.save_for_backward(logits, labels, stats)
        return stats[0]

    @staticmethod
    def backward(ctx, g):
        logits, labels, stats = ctx.saved_tensors
        B, C = logits.shape[:2]
        V = logits.numel() // (B * C)
        gz = torch.empty_like(logits)
        gup = g.contiguous().float().reshape(1)
        _lib.call("dp_dice_ce_bwd", _p(logits), _p(labels), _LABEL_KIND[labels.dtype], B, C, V, _p(stats), _p(gup), _p(gz), _stream())
        return gz, None, None, None, None, None


def dice_ce(logits, labels, smooth_nr=1e-5, smooth_dr=1e-5, lambda_dice=1.0, lambda_ce=1.0):
    return DiceCE.apply(logits, labels, smooth_nr, smooth_dr, lambda_dice, lambda_ce)


def dose_score(pred, gt, mask, scale=70.0):
    """Validation metric of train_light_pyfer.py:166-172: post-process (zero where mask < 1 or pred < 0), then
    scale * mean |pred - gt| over mask > 0 (evaluate_openKBP.get_3D_Dose_dif).  No gradient; 0-dim device tensor."""
    _chk_dev(pred, gt, mask)
    pred, gt, mask = pred.detach().contiguous().float(), gt.contiguous().float(), mask.contiguous().float()
    n = pred.numel()
    ws = torch.empty((_lib.lib().dp_masked_l1_ws_elems(n),), dtype=torch.float32, device=pred.device)
    out = torch.empty((3,), dtype=torch.float32, device=pred.device)
    _lib.call("dp_masked_l1_fwd", _p(pred), _p(gt), _p(mask), n, _p(ws), _p(out), 1, _stream())
    return out[2] * scale


def dose_postprocess(pred, mask, scale=70.0):
    """pred[(mask < 1) | (pred < 0)] = 0; x scale (train_light_pyfer.py:166-172)."""
    _chk_dev(pred, mask)
    pred, mask = pred.detach().contiguous().float(), mask.contiguous().float()
    out = torch.empty_like(pred)
    _lib.call("dp_dose_postprocess", _p(pred), _p(mask), _p(out), pred.numel(), float(scale), _stream())
    return out


# ------------------------------------------------------------------------------------------------ launch-thread economy
def _direct_apply():
    """torch.autograd.Function.apply is a PYTHON classmethod: it binds default arguments for setup_context-style Functions, asks functorch
    whether a transform is active and walks every argument through _functorch.utils.unwrap_dead_wrappers before it reaches the C++
    THPFunction_apply (3-4 us per call; ~380 applications per training step, tools/host_profile.py).  None of that applies here (no
    setup_context, no functorch transforms over raw-pointer kernels), so every Function of this module calls the C++ entry point directly:
    same autograd graph, same results.  DOSE_HIP_PY_APPLY=1 keeps the Python classmethod (A/B)."""
    if os.environ.get("DOSE_HIP_PY_APPLY"):
        return
    base = torch.autograd.Function
    for obj in list(globals().values()):
        if isinstance(obj, type) and issubclass(obj, base) and obj is not base and "apply" not in obj.__dict__:
            try:
                obj.apply = super(base, obj).apply
            except Exception:      # (a torch build without the C classmethod: keep the stock path)
                return


_direct_apply()
