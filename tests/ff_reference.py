"""The feed-forward operators (closerlook3d_amd/feed_forward.py) in 64 bits, on point-major rows, with bounds on how far an
evaluation in f32 with one rounding to the tensors' type may be from them.

A bound follows the formula: every f32 sum of n products is off by at most (n + 8) 2^-24 of the sum of their magnitudes, a
rounding to the type by half a step of the value (and half the smallest subnormal), and both travel through what comes after by
its slope."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest subnormal (bf16 and f32: nothing at these magnitudes)."""
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def rounding(v, dtype):
    return half_step(dtype) * v.abs() + tiny(dtype)


# slope of the activations is at most 1.13, its change at most 0.8 per unit (GELU; SiLU 1.1 and 0.5)
def activation(kind, g):
    if kind == 'silu':
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if kind == 'gelu':
        c = 0.5 * (1.0 + torch.erf(g / math.sqrt(2.0)))
        return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    return torch.relu(g), (g > 0).to(g.dtype)


def ffn(x, wg, wu, wd, kind, dy=None, dtype=torch.float32, inner=None):
    """{'y', 'dx', 'dwg', 'dwu', 'dwd'} -> (value, bound).  Arguments in 64 bits, rows (R, C); dtype: of the tensors; inner: what
    enters a product is rounded to (the tensors' type, or bfloat16 under precision 'bf16')."""
    inner = inner or dtype
    lossy_in = inner != dtype

    def entering(v):  # an operand and how far its rounding moved it
        e = rounding(v, inner) if lossy_in else torch.zeros_like(v)
        return v, e

    def prod(a, ea, b, eb, n):  # a b^T with operand errors, n terms
        s = a.abs() @ b.abs().t()
        return a @ b.t(), (n + 8) * U32 * s + ea @ b.abs().t() + a.abs() @ eb.t() + ea @ eb.t()

    R, C = x.shape
    H = wg.shape[0]
    (x, ex), (wg, eg_), (wu, eu_) = entering(x), entering(wg), entering(wu)
    g, eg = prod(x, ex, wg, eg_, C)
    u, eu = prod(x, ex, wu, eu_, C)
    a, slope = activation(kind, g)
    ea = 1.13 * eg + 8 * U32 * a.abs()
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + ea * eu + 2 * U32 * h.abs()
    out = {}
    if wd is None:
        out['y'] = (h, eh + rounding(h, dtype))
    else:
        wd, ed = entering(wd)
        ehr = eh + (rounding(h, inner) if inner != torch.float32 else 0.0)
        y, ey = prod(h, ehr, wd, ed, H)
        out['y'] = (y, ey + rounding(y, dtype))
    if dy is None:
        return out
    if wd is None:
        dh, edh = dy, torch.zeros_like(dy)
    else:
        dy, edy = entering(dy)
        dh, edh = prod(dy, edy, wd.t(), ed.t(), C)
    es = 0.8 * eg + 16 * U32 * (1.0 + g.abs())
    if kind == 'relu':
        es = (g.abs() <= eg).to(g.dtype)  # the side of the corner is not known there
    dg, du = dh * u * slope, dh * a
    edg = edh * (u * slope).abs() + (dh * slope).abs() * eu + (dh * u).abs() * es + edh * eu + 4 * U32 * dg.abs()
    edu = edh * a.abs() + dh.abs() * ea + edh * ea + 4 * U32 * du.abs()
    if inner != torch.float32:
        edg, edu = edg + rounding(dg, inner), edu + rounding(du, inner)
    p, ep = prod(dg, edg, wg.t(), eg_.t(), H)
    q, eq = prod(du, edu, wu.t(), eu_.t(), H)
    out['dx'] = (p + q, ep + eq + H * U32 * (dg.abs() @ wg.abs()) + rounding(p + q, dtype))
    for name, d, e in (('dwg', dg, edg), ('dwu', du, edu)):
        w, ew = prod(d.t(), e.t(), x.t(), ex.t(), R)
        out[name] = (w, ew + rounding(w, dtype))
    if wd is not None:
        w, ew = prod(dy.t(), edy.t(), h.t(), ehr.t(), R)
        out['dwd'] = (w, ew + rounding(w, dtype))
    return out


def words(seed, offset, count):
    """Philox 4x32 with ten rounds by numpy's 64-bit products: word i is number i % 4 of block offset + i / 4."""
    at = np.arange((count + 3) // 4, dtype=np.uint64) + np.uint64(offset % 2 ** 64)
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    a, b = at & low, at >> shift
    c, d = np.zeros_like(a), np.zeros_like(a)
    for r in range(10):
        k0, k1 = (seed + r * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF
        u, w = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (w >> shift) ^ b ^ np.uint64(k0), w & low, (u >> shift) ^ d ^ np.uint64(k1), u & low
    return np.stack([a, b, c, d], 1).reshape(-1)[:count]


def keep(seed, offset, p, shape):
    """True where an element stays."""
    n = math.prod(shape)
    return torch.from_numpy(words(seed, offset, n) >= np.uint64(int(p * 2 ** 32))).reshape(shape)


def _hat(v, kind, eps):
    if kind == 'none':
        return v, torch.ones_like(v[:, :1]), 0.0
    mean = v.mean(1, keepdim=True) if kind == 'layer' else 0.0
    inv = 1.0 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + eps)
    hat = (v - mean) * inv
    # a mean of C values: (C + 8) roundings of their magnitudes; the deviation's relative error is of that order too
    k = (v.shape[1] + 32) * U32
    return hat, inv, k * (hat.abs() + inv * v.abs().mean(1, keepdim=True)) + 2 * U32 * inv * v.abs()


def _hat_grad(dhat, e, hat, ehat, inv, kind):
    """Gradient through a norm, and its bound, for the gradient `dhat` (off by e) of the normalised rows."""
    if kind == 'none':
        return dhat, e
    C = dhat.shape[1]
    k = (C + 32) * U32
    m = (dhat * hat).mean(1, keepdim=True)
    em = (k * (dhat * hat).abs() + e * hat.abs() + dhat.abs() * ehat).mean(1, keepdim=True)
    d = dhat - hat * m
    ed = e + ehat * m.abs() + hat.abs() * em + ehat * em + 4 * U32 * (dhat.abs() + (hat * m).abs())
    if kind == 'layer':
        d = d - dhat.mean(1, keepdim=True)
        ed = ed + (k * dhat.abs() + e).mean(1, keepdim=True) + 2 * U32 * dhat.abs()
    return d * inv, ed * inv * (1 + k) + 2 * k * (d * inv).abs()


def norm(x, y=None, weight=None, bias=None, gate=None, scale=1.0, kind='rms', eps=1e-6, mask=None, p=0.0, next_kind=None,
         next_weight=None, next_bias=None, dout=None, dnext=None, dtype=torch.float32, clouds=1):
    """{'out', 'next', 'dx', 'dy', 'dweight', ...} -> (value, bound), rows in 64 bits.  mask: True where an element stays; gate (C,)
    or (clouds, C)."""
    res = {}
    R, C = x.shape
    one = torch.ones((C,), dtype=x.dtype, device=x.device)
    o, eo = x, torch.zeros_like(x)
    if y is not None:
        hat1, inv1, e1 = _hat(y, kind, eps)
        w, b = one if weight is None else weight, 0 * one if bias is None else bias
        m = torch.ones_like(x) if mask is None else mask.to(x.dtype).to(x.device) / (1.0 - p)
        g = one.expand(R, C) if gate is None else gate.expand(R, C) if gate.dim() == 1 else gate.repeat_interleave(R // clouds, 0)
        n = hat1 * w + b
        en = e1 * w.abs() + 3 * U32 * ((hat1 * w).abs() + b.abs())
        o = scale * x + g * (n * m)
        eo = g.abs() * m * en + 4 * U32 * ((scale * x).abs() + (g * n * m).abs())
        res['out'] = (o, eo + rounding(o, dtype))
    if next_kind is not None:
        hat2, inv2, e2 = _hat(o, next_kind, eps)
        e2 = e2 + inv2 * eo + (hat2.abs() + 1) * (inv2 * eo).mean(1, keepdim=True) + hat2.abs() * (hat2 * inv2 * eo).abs().mean(1, keepdim=True)
        w2, b2 = one if next_weight is None else next_weight, 0 * one if next_bias is None else next_bias
        v = hat2 * w2 + b2
        res['next'] = (v, e2 * w2.abs() + 3 * U32 * ((hat2 * w2).abs() + b2.abs()) + rounding(v, dtype))
    if dout is None and dnext is None:
        return res

    def total(v, e, per_cloud=False):  # a sum over the rows
        s = (R + 8) * U32 * v.abs() + e
        v, s = (v.reshape(clouds, -1, C).sum(1), s.reshape(clouds, -1, C).sum(1)) if per_cloud else (v.sum(0), s.sum(0))
        return v, s + rounding(v, dtype)

    d = torch.zeros_like(x) if dout is None else dout
    ed = torch.zeros_like(x)
    if dnext is not None:
        res['dnext_weight'] = total(dnext * hat2, dnext.abs() * e2)
        res['dnext_bias'] = total(dnext, ed)
        t, et = _hat_grad(dnext * w2, U32 * (dnext * w2).abs(), hat2, e2, inv2, next_kind)
        d, ed = d + t, et + U32 * (d.abs() + t.abs())
    if y is None:
        res['dx'] = (d, ed + rounding(d, dtype))
        return res
    dx = scale * d
    res['dx'] = (dx, abs(scale) * ed + U32 * dx.abs() + rounding(dx, dtype))
    dm, edm = d * m, ed * m + U32 * (d * m).abs()
    res['dgate'] = total(dm * n, edm * n.abs() + dm.abs() * en, gate is not None and gate.dim() == 2)
    dn, edn = dm * g, edm * g.abs() + U32 * (dm * g).abs()
    res['dweight'] = total(dn * hat1, edn * hat1.abs() + dn.abs() * e1)
    res['dbias'] = total(dn, edn)
    t, et = _hat_grad(dn * w, edn * w.abs() + U32 * (dn * w).abs(), hat1, e1, inv1, kind)
    res['dy'] = (t, et + rounding(t, dtype))
    return res


def check(got, want, what):
    """Every element within its bound; a bound of 0 with an exact value means equal."""
    value, bound = want
    got = got.double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got - value).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), "of", bad.numel(), "worst", float((off / bound.clamp_min(1e-300))[bad].max()),
                                 [int(i) for i in bad.nonzero()[0]], float(got[bad][0]), float(value[bad][0]))
