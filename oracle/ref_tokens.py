"""Float64 restatement of the token operators (rotary positions over grid axes, per-head norm of queries and keys, sliding-window
attention) with elementwise bounds of what a kernel of a given storage type may be off.  Test infrastructure only.

Bounds: `u` is half a step of the storage type relative to the value (one rounding), E = 2^-24 that of the fp32 arithmetic."""
import math

import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def angles(positions, sections, d, base=10000.0):
    """[.., N, 1, d / 2] float64; pairs behind the sections have angle 0."""
    cols = [positions[..., a:a + 1].double() * base ** (-torch.arange(n, dtype=torch.float64, device=positions.device) / n) for a, n in enumerate(sections) if n]
    ang = torch.cat(cols, -1)
    ang = torch.nn.functional.pad(ang, (0, d // 2 - ang.shape[-1]))
    return ang.unsqueeze(-2)


def rotary(x, positions, sections, base=10000.0, interleaved=False):
    """x [B, N, heads, d] float64."""
    ang = angles(positions, sections, x.shape[-1], base)
    c, s = ang.cos(), ang.sin()
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    y0, y1 = a * c - b * s, a * s + b * c
    return torch.stack((y0, y1), -1).flatten(-2) if interleaved else torch.cat((y0, y1), -1)


def pair_size(x, interleaved=False):
    """|a| + |b| of the pair every channel belongs to: what the rounding errors of a turn are proportional to."""
    half = x.shape[-1] // 2
    if interleaved:
        m = x[..., 0::2].abs() + x[..., 1::2].abs()
        return m.repeat_interleave(2, -1)
    m = x[..., :half].abs() + x[..., half:].abs()
    return torch.cat((m, m), -1)


def head_norm(x, w, b, eps=1e-5):
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    return (x - mean) * (var + eps).rsqrt() * w + b


def seen(B, Nq, Nk, left, right, sinks, start, lengths, device):
    j = torch.arange(Nk, device=device).view(1, 1, Nk)
    start = torch.as_tensor(start, device=device).long().reshape(-1, 1).expand(B, 1)
    p = (start + torch.arange(Nq, device=device)).unsqueeze(-1)
    n = (torch.full((B,), Nk, device=device) if lengths is None else lengths.to(device).long().clamp(0, Nk)).view(B, 1, 1)
    m = (j < n) & (p >= 0) & (p < n)
    if right is not None:
        m = m & (j <= p + right)
    if left is not None:
        m = m & ((j >= p - left) | (j < sinks))
    return m          # [B, Nq, Nk]


def window(q, k, v, g=None, left=None, right=None, sinks=0, start=0, lengths=None, scale=None, dtype=torch.float32, in_err=0.0):
    """Everything in float64 from the exact values of the (already rounded) operands.  Returns [(value, bound)] of out and, with g, of dq,
    dk, dv.  in_err: relative error that q and k themselves may carry (a rounding between two fused steps).

    Bounds (u: half step of `dtype`, 0 for fp32 inside because every fp32 product and sum is counted by E):
      score: s = scale q.k in fp32: |ds| <= scale ((d + 4) E + 2 in_err) |q|.|k|, and 4 E |s| for the change of base and the exponent
      p: relative 2 max|ds| (numerator and normaliser) + 16 E + u (rounded for the second product)
      out: u |out| + (rel p + Nk E) sum p |v|
      lse adds nothing new to p in the backward pass; delta = dO.O with O stored: |ddelta| <= |dO|.(bound of out) + d E |dO|.|O|
      dS: (rel p) |dS| + p scale ((d + 2) E |dO|.|V| + |ddelta|) + u |dS|
      p and dS below 2^-14 are fp16 subnormals, steps of 2^-24 apart: each may be off by half of one, 2^-25, whatever its size
      sums over queries / keys: (rows) E of the absolute terms."""
    u = half_step(dtype)
    ui = u if dtype != torch.float32 else 0.0
    B, Nq, heads, d = q.shape
    Nk, kv = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    group = heads // kv
    q, k, v = q.double(), k.double(), v.double()
    m = seen(B, Nq, Nk, left, right, sinks, start, lengths, q.device)
    okq, okk = m.any(2)[:, :, None, None], m.any(1)[:, :, None, None]
    q, k, v = torch.where(okq, q, 0.0), torch.where(okk, k, 0.0), torch.where(okk, v, 0.0)      # (what is never seen may hold anything)
    Q, K, V = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(group, 1), v.transpose(1, 2).repeat_interleave(group, 1)
    mm = m.unsqueeze(1)
    s = (Q @ K.transpose(-1, -2)) * scale
    es = scale * ((d + 4) * E + 2 * in_err) * (Q.abs() @ K.abs().transpose(-1, -2)) + 4 * E * s.abs()
    s = s.masked_fill(~mm, -math.inf)
    top = s.amax(-1, keepdim=True) if Nk else s.new_zeros(B, heads, Nq, 1)
    p = (s - torch.where(top.isinf(), 0.0, top)).exp()
    L = p.sum(-1, keepdim=True)
    p = p / torch.where(L > 0, L, 1.0)
    rel = 2 * torch.where(mm, es, 0.0).amax(-1, keepdim=True) + 16 * E + ui if Nk else L + 0.0
    rel = rel + 8 * E * s.masked_fill(~mm, 0.0).abs().amax(-1, keepdim=True) if Nk else rel
    out = p @ V
    sub = (2.0 ** -25 if dtype == torch.float16 else 0.0) * mm.double()
    eo = u * out.abs() + (rel + Nk * E) * (p @ V.abs()) + sub @ V.abs()
    res = [(out.transpose(1, 2), eo.transpose(1, 2))]
    if g is None:
        return res
    G = torch.where(okq, g.double(), 0.0).transpose(1, 2)
    dP = G @ V.transpose(-1, -2)
    delta = (G * out).sum(-1, keepdim=True)
    ed = (G.abs() * eo).sum(-1, keepdim=True) + d * E * (G.abs() * out.abs()).sum(-1, keepdim=True)
    dS = p * (dP - delta) * scale
    edS = (rel + ui) * dS.abs() + p * scale * ((d + 2) * E * (G.abs() @ V.abs().transpose(-1, -2)) + ed) + sub
    dQ, dK, dV = dS @ K, dS.transpose(-1, -2) @ Q, p.transpose(-1, -2) @ G
    n = Nq * group
    eQ = u * dQ.abs() + (edS + (Nk * E + in_err) * dS.abs()) @ K.abs()
    eK = (edS + (n * E + in_err) * dS.abs()).transpose(-1, -2) @ Q.abs()
    eV = ((rel + ui + n * E) * p + sub).transpose(-1, -2) @ G.abs()
    fold = lambda t: t.view(B, kv, group, Nk, d).sum(2).transpose(1, 2)  # noqa: E731
    dK, dV = fold(dK), fold(dV)
    return res + [(dQ.transpose(1, 2), eQ.transpose(1, 2)), (dK, u * dK.abs() + fold(eK)), (dV, u * dV.abs() + fold(eV))]
