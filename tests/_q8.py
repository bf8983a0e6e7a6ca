"""The 8-bit linear layers' operators from their formulas, in 64 bits, and how far the kernels may be off.

What a tolerance counts: a code is the formula's, but for the last bits of the quotient here (2^-45) at a tie;
a sum of k squares in 32 bits, all positive, is off by at most one rounding for each addition that an element goes
through; an integer sum turned to fp32, the two scales and the two additions are a rounding of 2^-24 each; a result
in fp16 is off by 2^-11 of its value or half of the smallest step, 2^-25."""
import torch

TOP = 127.0


def quantise(y):
    """fp64 rows [m, k] -> (codes, distance of 127 y / max from the nearest tie, scales)."""
    bad = ~torch.isfinite(y).all(dim=1)
    z = torch.where(bad[:, None], torch.zeros_like(y), y)
    top = z.abs().amax(dim=1)
    q = z * (TOP / torch.where(top > 0, top, torch.ones_like(top)))[:, None]
    tie = (q.abs() - torch.floor(q.abs()) - 0.5).abs()
    return torch.round(q), tie, torch.where(bad, torch.nan, top / TOP)


def norm(s, gamma, eps):
    s = s.double()
    return s * torch.rsqrt((s * s).mean(dim=1, keepdim=True) + eps) * gamma.double()


def check_rows(y, codes, scales, values=None, k=1, additions=0):
    """Codes, scales and values against fp64 rows y."""
    want, tie, scale = quantise(y)
    c = codes.double()
    off = (c - want).abs()
    assert bool(((off == 0) | ((off == 1) & (tie < 2.0 ** -40))).all()), f"codes off by {float(off.max())}"
    assert torch.equal(torch.isnan(scales.double()), torch.isnan(scale))
    fine = ~torch.isnan(scale)
    rel = (additions / 2 + 6) * 2.0 ** -24
    assert bool(((scales.double() - scale).abs()[fine] <= rel * scale[fine]).all())
    if values is not None:
        v = c * scales.double()[:, None]
        assert bool(torch.isnan(values[~fine]).all())
        err = (values.double() - v).abs()[fine]
        assert bool((err <= v.abs()[fine] * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all())


def linear(x, xs, w, ws):
    """The scaled sums, exact in fp64 (53 bits hold them)."""
    return (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()


def check_linear(y, x, xs, w, ws, bias=None, residual=None):
    v = linear(x, xs, w, ws)
    size = v.abs()
    for t in (bias, residual):
        if t is not None:
            v = v + t.double()
            size = size + t.double().abs()
    _near(y, v, v.abs() * 2.0 ** -11 + size * 2.0 ** -21)


def check_gated(y, x, xs, w, ws):
    n = w.shape[0] // 2
    g, u = linear(x, xs, w[:n], ws[:n]), linear(x, xs, w[n:], ws[n:])
    v = g * torch.sigmoid(g) * u
    # d silu(g) / silu(g) = (1 + g (1 - sigmoid(g))) dg / g, g off by 3 roundings; exp off by 2 units (2^-22)
    _near(y, v, v.abs() * (2.0 ** -11 + 2.0 ** -21 * (2.0 + g.abs())))


def _near(y, v, tol):
    y = y.double()
    assert torch.equal(torch.isnan(y), torch.isnan(v))
    top = 65520.0  # from here on fp16 rounds to infinity
    big = v.abs() > top * (1 + 2.0 ** -10)
    assert bool((torch.isinf(y) | torch.isnan(y) | ~big).all())
    fine = torch.isfinite(v) & (v.abs() < top * (1 - 2.0 ** -10)) & ~torch.isnan(v)
    err = (y - v).abs()[fine] - (tol[fine] + 2.0 ** -25)
    assert err.numel() == 0 or float(err.max()) <= 0, f"off by {float(err.max()):.3g} more than allowed"


def padded(m, k, dtype, device, extra=0, fill=0):
    """A [m, k] view whose rows start at multiples of 16 elements, `extra` 16s further apart than needed."""
    ld = -(-k // 16) * 16 + 16 * extra
    return torch.full((m, ld), fill, dtype=dtype, device=device)[:, :k]


def rand_codes(m, k, gen, device, lo=-127, hi=127, extra=0):
    c = padded(m, k, torch.int8, device, extra, fill=99)
    c.copy_(torch.randint(lo, hi + 1, (m, k), generator=gen, device=device, dtype=torch.int16).to(torch.int8))
    return c
