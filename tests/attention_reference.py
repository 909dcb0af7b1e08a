"""
Attention in 64 bits with elementwise bounds on what a kernel may be off by, for the tests of the packed
and the paged attention.

u = 2^-24 (f32 rounding), t = half a step of the tensors' type (0 extra for f32: its roundings are the u
terms).  A kernel computes
  s = scale q.k           d + 2 roundings of terms that sum to at most S = scale |q|.|k|:  ds = (d + 2) u S
  w = 2^(s c - m)         relative error of w: ds + |s| and |m| roundings of the scaled logs, 4 u for 2^x
  o = sum w v / sum w     numerator and denominator: twice w's error, n u for either sum, t for w
                          rounded to the type ahead of the product, t for the result
and the gradients analogously (`gradients`).  f16 has no exponent below 2^-14: a number smaller than that is
rounded to a multiple of 2^-24, off by at most z = 2^-25 whatever its size.  That holds for the result, for a
weight (forward: the weights are taken against a reference no larger than the row's maximum, so their sum
is at least 1 and z bounds the normalised weight's error too) and for gs = w (gp - delta) ahead of its
products: z per visible pair.  The bounds are first order; the factor 1.01 covers the
products of the terms.
"""
import torch

U = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def tiny(dtype):
    return 2.0**-25 if dtype == torch.float16 else 0.0


def weights(q, k, offset, causal, scale):
    """q Tq x D, k Tk x D in 64 bits -> (w, relative bound on w Tq x 1, visible)"""
    d = q.shape[1]
    s = q @ k.T * scale
    spread = (q.abs() @ k.abs().T) * scale
    see = torch.ones_like(s, dtype=torch.bool)
    if causal:
        see = torch.arange(k.shape[0])[None, :] <= offset + torch.arange(q.shape[0])[:, None]
    s = s.masked_fill(~see, float("-inf"))
    m = s.max(-1, keepdim=True)[0]
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    w = torch.where(total > 0, e / total.clamp_min(1e-300), torch.zeros_like(e))
    big = torch.where(see, spread, torch.zeros_like(spread)).max(-1, keepdim=True)[0] if k.shape[0] else total
    rel = 2 * ((d + 2) * U * big + 8 * big * U + 8 * U) + 2 * k.shape[0] * U
    return w, rel, see


def attend(q, k, v, offset, causal, scale, dtype):
    """one head -> (out, elementwise bound)"""
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    w, rel, see = weights(q, k, offset, causal, scale)
    t, z = half_step(dtype), tiny(dtype)
    out = w @ v
    return out, 1.01 * ((rel + t) * (w @ v.abs()) + z * (see.double() @ v.abs()) + (t + 2 * U) * out.abs() + z) + 1e-30


def gradients(q, k, v, g, causal, scale, dtype):
    """one head of a packed sequence -> out, gq, gk, gv and a bound for each"""
    d, n, t, z = q.shape[1], q.shape[0], half_step(dtype), tiny(dtype)
    w, rel, see = weights(q, k, 0, causal, scale)
    see = see.double()
    out = w @ v
    e_out = 1.01 * ((rel + t) * (w @ v.abs()) + z * (see @ v.abs()) + (t + 2 * U) * out.abs() + z)
    gp = g @ v.T
    e_gp = (d + 2) * U * (g.abs() @ v.abs().T)
    delta = (g * out).sum(-1, keepdim=True)
    # (delta is formed from out and what its rounding took away, itself rounded to the type)
    e_whole = 1.01 * ((rel + t) * (w @ v.abs()) + z * (see @ v.abs()) + (t * t + 2 * U) * out.abs() + z)
    e_delta = (g.abs() * e_whole).sum(-1, keepdim=True) + (d + 2) * U * (g * out).abs().sum(-1, keepdim=True)
    gs = w * (gp - delta)
    e_gs = w * (e_gp + e_delta + 2 * U * (gp.abs() + delta.abs())) + (rel + t) * gs.abs() + z * see
    gv = w.T @ g
    e_gv = ((rel + t + n * U) * w + z * see).T @ g.abs() + t * gv.abs() + z
    gq = gs @ k * scale
    e_gq = (e_gs @ k.abs() + n * U * (gs.abs() @ k.abs())) * scale + (t + 3 * U) * gq.abs() + z
    gk = gs.T @ q * scale
    e_gk = (e_gs.T @ q.abs() + n * U * (gs.abs().T @ q.abs())) * scale + (t + 3 * U) * gk.abs() + z
    return [out, gq, gk, gv], [1.01 * e + 1e-30 for e in (e_out, e_gq, e_gk, e_gv)]


def packed(q, k, v, lens, causal, scale=None, g=None):
    """q T x Hq x D ... of any type, rows behind sum(lens) zeros -> values and bounds in 64 bits, on the CPU"""
    dtype, D = q.dtype, q.shape[2]
    scale = D**-0.5 if scale is None else scale
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    like = [q, q, k, v] if g is not None else [q]
    vals, bounds = [torch.zeros_like(x) for x in like], [torch.zeros_like(x) for x in like]
    a = 0
    for n in lens:
        b = a + n
        for h in range(q.shape[1] if n else 0):
            c = h // (q.shape[1] // k.shape[1])
            if g is None:
                r, e = attend(q[a:b, h], k[a:b, c], v[a:b, c], 0, causal, scale, dtype)
                r, e = [r], [e]
            else:
                r, e = gradients(q[a:b, h], k[a:b, c], v[a:b, c], g[a:b, h].detach().cpu().double(), causal, scale,
                                 dtype)
            for i, (x, y) in enumerate(zip(r, e)):
                at = h if i < 2 else c
                vals[i][a:b, at] += x
                bounds[i][a:b, at] += y
        a = b
    return vals, bounds


def check(got, want, bound, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3e} above its bound, at {(over == over.max()).nonzero()[0].tolist()}"
