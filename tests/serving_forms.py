"""The serving operators in 64 bits, and how far a kernel's 32- and 16-bit arithmetic may be from them.

A kernel forms a score in 32 bits, takes 2^x, rounds the probability to fp16, sums products in 32 bits and rounds the output to
fp16.  Bounds (u = half a step of the type: fp16 2^-11, fp32 2^-24), worst case, per output element:
  score:       |ds| <= d = (D + 8) u32 max_j sum_c |q_c k_c| scale + u32 8 max|s| + cap * 2^-20 (tanh from two hardware
               functions of 1 ulp each: 2 / (e + 1) and e are off by at most a few 2^-23, times the cap; 0 without a cap)
  probability: relative 2 d + 2^-20 (both its exponent and the maximum's; exp2 to 1 ulp), then u16, or 2^-25 absolute where it is
               below fp16's normal range; the row's sum has at least the value 1
  output:      (u16 + 4 d + 2^-19) A + u16 |o| + N 2^-25 max|v|,  A = sum p |v|: the normaliser carries the same relative error
  lse:         2 d + 2^-20 (1 + |lse|)
"""
import math

import torch

U16, U32 = 2.0 ** -11, 2.0 ** -24


def rows_form(q, k, v, see, scale, softcap=0.0, slope=None, gap=None):
    """One head in 64 bits: q [R, D], k, v [N, D], see [R, N].  Returns o, lse, p, and the bounds of the first two and of a
    relative probability.  Values no row sees are left out; where a row sees an infinite or undefined value o is not finite."""
    q, k = q.double(), k.double()
    any_see = see.any(0)
    k = torch.where(any_see[:, None], k, torch.zeros_like(k))
    # a key that only some rows see may hold anything for the others
    raw = torch.where(see, q @ k.T.contiguous(), torch.zeros((), dtype=torch.float64, device=q.device)) if torch.isfinite(k).all() else \
        torch.stack([torch.where(see[i], (q[i] * k).sum(1), torch.zeros((), dtype=torch.float64, device=q.device)) for i in range(q.shape[0])])
    s = raw * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slope is not None:
        s = s - float(slope) * gap.abs().double()
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    top = s.max(1, keepdim=True).values
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(s - top)
    z = e.sum(1, keepdim=True)
    p = e / torch.where(z > 0, z, torch.ones_like(z))
    o = torch.zeros(q.shape[0], q.shape[1], dtype=torch.float64, device=q.device)
    if v is not None:
        vd = v.double()
        clean = torch.where(torch.isfinite(vd), vd, torch.zeros_like(vd))
        o = p @ clean
        dirty = (~torch.isfinite(vd)).double()
        hit = see.double() @ dirty > 0
        amount = p @ clean.abs()
    lse = torch.log(z)[:, 0] + top[:, 0]
    lse = torch.where(see.any(1), lse, torch.full_like(lse, -math.inf))
    kf = torch.where(torch.isfinite(k), k, torch.zeros_like(k)).abs()
    qf = torch.where(torch.isfinite(q), q, torch.zeros_like(q)).abs()
    mag = (qf @ kf.T.contiguous()).max().item() * scale if k.numel() else 0.0
    most = s[see].abs().max().item() if see.any() else 0.0
    d = (q.shape[1] + 8) * U32 * mag + 8 * U32 * most + (softcap * 2.0 ** -20 if softcap else 0.0)
    tol_lse = 2 * d + 2.0 ** -20 * (1 + lse.abs())
    if v is None:
        return None, lse, p, None, tol_lse, 2 * d + 2.0 ** -20
    tol = (U16 + 4 * d + 2.0 ** -19) * amount + U16 * o.abs() + k.shape[0] * 2.0 ** -25 * (clean.abs().max().item() if clean.numel() else 0.0) + 2.0 ** -25
    o = torch.where(hit, torch.full_like(o, math.nan), o)
    return o, lse, p, tol, tol_lse, 2 * d + 2.0 ** -20


def check_rows(got, want, tol, what):
    """|got - want| <= tol where want is finite; where it is not, got must not be either."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: {int((torch.isfinite(got) != fine).sum())} values are finite in one and not in the other"
    over = torch.where(fine, (got - want).abs() - tol, torch.zeros_like(want))
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {int((over > 0).sum())} values off, one by {worst:.3e} beyond its bound"


def prompt_see(n, S, device, prefix=None, docs=None):
    """[S, S]: which token (column) each row sees."""
    i, j = torch.arange(S, device=device)[:, None], torch.arange(S, device=device)[None]
    see = j <= i
    if prefix is not None:
        see = see | (j < prefix)
    see = see & (i < n) & (j < n)
    if docs is not None:
        see = see & (docs[:, None] == docs[None]) & (docs[:, None] >= 0)
    return see


def nibbles(p):
    return torch.stack([p >> 4, p & 15], -1).flatten(-2).to(torch.int32)


def joined(hi, mid, last):
    return ((hi.to(torch.int32) << 8) | (nibbles(mid) << 4) | nibbles(last)).to(torch.int16).view(torch.half)


def plane_tokens(cache, layer, b, h, n):
    """(k, v) fp16 [n, D] that the planes of a RaggedGQACache hold at the first n places of (sequence, KV head)."""
    kp, vp = cache.k_planes[layer], cache.v_planes[layer]
    D = cache.head_dim
    k = joined(*(p[b, h] for p in kp)).permute(0, 2, 1).reshape(-1, D)[:n]
    v = joined(*(p[b, h] for p in vp))[:n]
    return k, v


def cached_tokens(cache, layer, b, h):
    """(k, v) fp16 [length, D]: the planes, then the rest buffer."""
    n = int(cache.seq_lens[layer][b])
    f = n // 64 * 64
    k, v = plane_tokens(cache, layer, b, h, f)
    return torch.cat([k, cache.restk[layer][b, :n - f, h]]), torch.cat([v, cache.restv[layer][b, :n - f, h]])
