"""Plain 64-bit forms of the language-model client operators and the error
bounds their tests use (CPU, float64).

A product of k terms summed in float32 in any order is off by at most
k * 2^-24 * sum |a||b| to first order.  Where a float32 or fp16 operand is fed
to the bf16 matrix units as two bf16 terms (nearest, then the rest), the rest's
own rounding leaves 2^-18 of the operand, and the product of the two rests,
left out, is at most 2^-18 of the product: three such per product stay below
2^-16.  ``PROD`` is that; the final rounding adds eps / 2 of the result.
"""
from __future__ import annotations

import torch

PROD = 2.0 ** -16
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def segments(offsets, slots, tokens):
    """[(first, last, slot)] of the tokens that have one."""
    o = [min(max(int(v), 0), tokens) for v in offsets]
    return [(o[s], o[s + 1], int(c)) for s, c in enumerate(slots) if int(c) >= 0 and o[s + 1] > o[s]]


def d(t):
    return t.detach().cpu().double()


def product(a, ea, b, eb):
    """a @ b and a bound of its error, for operands known up to ea and eb."""
    k = a.shape[1]
    c = k * U + PROD
    err = a.abs() @ eb + ea @ b.abs() + ea @ eb + c * ((a.abs() + ea) @ (b.abs() + eb))
    return a @ b, err


def adapter(base, x, A, B, offsets, slots, scale, dtype, dy=None, dx_base=None):
    """dict of (value, error bound) for out and, with dy, dx, dA, dB."""
    T = x.shape[0]
    x, A, B = d(x), d(A), d(B)
    n, r, K = A.shape
    M = B.shape[1]
    out = d(base).clone() if base is not None else torch.zeros(T, M, dtype=torch.float64)
    eout = torch.zeros_like(out)
    res = {}
    if dy is not None:
        dy = d(dy)
        dx = d(dx_base).clone() if dx_base is not None else torch.zeros(T, K, dtype=torch.float64)
        edx = torch.zeros_like(dx)
        dA, eA = torch.zeros(n, r, K, dtype=torch.float64), torch.zeros(n, r, K, dtype=torch.float64)
        dB, eB = torch.zeros(n, M, r, dtype=torch.float64), torch.zeros(n, M, r, dtype=torch.float64)
    s = abs(scale)
    for a, b, c in segments(offsets, slots, T):
        xs, Ac, Bc = x[a:b], A[c], B[c]
        zero = torch.zeros_like
        h, eh = product(xs, zero(xs), Ac.T.contiguous(), zero(Ac.T))
        y, ey = product(h, eh, Bc.T.contiguous(), zero(Bc.T))
        base_part = out[a:b].abs()
        out[a:b] += scale * y
        # scale as float32, the product with it and the sum: one rounding each
        eout[a:b] = s * ey + U * (3 * s * y.abs() + base_part + out[a:b].abs())
        if dy is not None:
            g = dy[a:b]
            z, ez = product(g, zero(g), Bc, zero(Bc))
            v, ev = product(z, ez, Ac, zero(Ac))
            base_part = dx[a:b].abs()
            dx[a:b] += scale * v
            edx[a:b] = s * ev + U * (3 * s * v.abs() + base_part + dx[a:b].abs())
            w, ew = product(z.T.contiguous(), ez.T, xs, zero(xs))
            dA[c] += scale * w
            eA[c] += s * ew + 4 * U * (s * w.abs() + dA[c].abs())
            w, ew = product(g.T.contiguous(), zero(g.T), h, eh)
            dB[c] += scale * w
            eB[c] += s * ew + 4 * U * (s * w.abs() + dB[c].abs())
    res["out"] = (out, eout + half_step(dtype) * (out.abs() + eout) + 1e-30)
    if dy is not None:
        res["dx"] = (dx, edx + half_step(dtype) * (dx.abs() + edx) + 1e-30)
        res["dA"], res["dB"] = (dA, eA + 1e-30), (dB, eB + 1e-30)
    return res


def token_slots(offsets, slots, T):
    out = torch.full((T,), -1, dtype=torch.int64)
    for a, b, c in segments(offsets, slots, T):
        out[a:b] = c
    return out


def embed_grad(dy, ids, n, V, offsets, slots, scale, padding=None):
    """(value, bound) of the (n, V, E) gradient; float32 sums of L terms in order
    and one product with the scale: (L + 2) * 2^-24 of the sum of magnitudes."""
    T, E = dy.shape
    ids = ids.cpu()
    slot = token_slots(offsets, slots, T) if offsets is not None else torch.zeros(T, dtype=torch.int64)
    keep = (slot >= 0) & (ids >= 0) & (ids < V)
    if padding is not None:
        keep &= ids != padding
    rows = (slot * V + ids)[keep]
    g = d(dy)[keep]
    val = torch.zeros(n * V, E, dtype=torch.float64).index_add_(0, rows, g) * scale
    mag = torch.zeros(n * V, E, dtype=torch.float64).index_add_(0, rows, g.abs()) * abs(scale)
    cnt = torch.bincount(rows, minlength=n * V).double()[:, None]
    return val.view(n, V, E), ((cnt + 3) * U * mag).view(n, V, E) + 1e-30


def logprobs(logits, targets, ignore=-100):
    """lse, logp, entropy and their bounds in 64 bits.

    With d = x - max: exp(d) in float32 through a rounded difference, a rounded
    product and a 1-ulp exp2 is off by (2 |d| + 4) * 2^-24 of itself; a thread adds
    at most V / 64 + 16 terms and 16 joins follow."""
    x = d(logits)
    V = x.shape[1]
    steps = V / 64 + 32
    m = x.max(dim=1, keepdim=True).values
    dd = torch.where(torch.isinf(x) & (x < 0), torch.zeros_like(x), x - m)
    p = torch.exp(x - m)
    s = p.sum(1, keepdim=True)
    p = p / s
    lse = (m + torch.log(s)).squeeze(1)
    t = targets.cpu()
    ok = (t >= 0) & (t < V)
    xt = x.gather(1, t.clamp(0, V - 1)[:, None]).squeeze(1)
    logp = torch.where(ok, xt - lse, torch.where(t == ignore, 0.0, float("nan")).double())
    a1, a2 = (p * dd.abs()).sum(1), (p * dd * dd).sum(1)
    ent = torch.log(s).squeeze(1) - (p * dd).sum(1)
    rel = U * (2 * a1 + 4 + steps)
    e_lse = rel + U * (2 * torch.log(s).squeeze(1).abs() + 2 * lse.abs() + m.squeeze(1).abs())
    e_logp = e_lse + U * (xt.abs() + 2 * logp.abs())
    e_ent = 2 * rel + U * (2 * a2 + (steps + 8) * a1 + 2 * torch.log(s).squeeze(1).abs() + 2 * ent.abs()) + rel * a1
    return dict(lse=lse, logp=logp, ent=ent, p=p, e_lse=e_lse, e_logp=e_logp, e_ent=e_ent, ok=ok, x=x)


def logits_grad(ref, targets, gl, ge, dtype):
    """(value, bound) of the logits' gradient."""
    p, lse, ent, ok, x = ref["p"], ref["lse"][:, None], ref["ent"][:, None], ref["ok"], ref["x"]
    gl = torch.where(ok, d(gl), torch.zeros(()).double())[:, None]
    g = -gl * p
    logp = torch.where(p > 0, x - lse, torch.zeros_like(x))
    # exp(x - lse) in float32: as exp(d), with the error of lse itself
    ep = p * (U * (2 * logp.abs() + 4 + 2 * lse.abs()) + ref["e_lse"][:, None])
    err = gl.abs() * ep + 3 * U * gl.abs() * p
    if ge is not None:
        ge = d(ge)[:, None]
        f = logp + ent
        g = g - ge * p * f
        err = err + ge.abs() * (ep * f.abs() + p * (U * (logp.abs() + 2 * lse.abs() + 4 * f.abs())
                                                    + ref["e_lse"][:, None] + ref["e_ent"][:, None])) \
            + U * (gl * p).abs()
    t = targets.cpu().clamp(0, x.shape[1] - 1)[:, None]
    g = g.scatter_add(1, t, gl)
    err = err + 2 * U * (g.abs() + gl.abs())
    # a value below the type's normal range is rounded by half its smallest step
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return g, err + half_step(dtype) * (g.abs() + err) + tiny + 2.0 ** -126 * (gl.abs() + 1)


def within(name, got, want, bound):
    got, want = d(got), want.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "%s: NaN in other places" % name
    err = (got - want).abs()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), "%s: infinities differ" % name
    bad = (err > bound) & ~nan & ~inf
    if bad.any():
        i = (err / bound).where(bad, torch.zeros_like(err)).argmax()
        raise AssertionError("%s: %d of %d beyond the bound, worst |%g - %g| = %g > %g"
                             % (name, int(bad.sum()), bad.numel(), got.flatten()[i], want.flatten()[i],
                                err.flatten()[i], torch.as_tensor(bound).expand_as(err).flatten()[i]))
