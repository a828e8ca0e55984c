"""Oracles in 64 bits of the 8-bit activations and of a gate layer's gradients at them, and bounds on
what fp32 evaluation may differ by.

Bounds: every quantity here but the sigmoid is a polynomial of its inputs. Evaluated in fp32 by n rounded
operations on any path from an input to the result, it is off by at most n * 2^-24 (to first order) times
the same polynomial at the inputs' absolute values, which ``mag`` tensors hold."""
import torch

EPS = 2.0 ** -24
GATE16, WALSH, MULTILINEAR = 0, 1, 2
F64 = torch.float64


def codes_of(x):
    """Codes [B, D], lo and step [B] of fp32 rows: the format is defined by its fp32 arithmetic."""
    x = x.float().cpu()
    lo, hi = x.amin(1), x.amax(1)
    span = hi - lo
    most = torch.full_like(span, 255.0)   # a tensor: 255.0 / span is torch's reciprocal times 255
    inv, step = most / span, span / most
    flat = ~(span > 0) | ~torch.isfinite(inv)
    inv[flat], step[flat] = 0.0, 0.0
    bad = ~torch.isfinite(x).all(1) | ~torch.isfinite(span)
    lo = torch.where(bad, torch.full_like(lo, float("nan")), lo)
    q = torch.round((x - x.amin(1, keepdim=True)) * inv[:, None])
    q[bad | flat] = 0
    step[bad] = 0.0
    return q, lo, step


def values_of(x):
    """What the codes stand for, in 64 bits."""
    q, lo, step = codes_of(x)
    return lo.to(F64)[:, None] + q.to(F64) * step.to(F64)[:, None]


def poly(kind, raw):
    """Coefficients {1, a, b, ab} of every output's node, their ``mag``, the function that takes their
    gradient back to the parameters, and its ``mag``. The coefficients are sums of terms of both signs
    (probabilities times basis entries, corners, Walsh weights): where those cancel, a coefficient is off by
    roundings of the terms' size and not of its own, so its ``mag`` is the sum of the terms' absolute values."""
    raw = raw.to(F64).cpu()
    if kind == GATE16:
        i = torch.arange(16)
        f00, f01, f10, f11 = (((i >> n) & 1).to(F64) for n in (3, 2, 1, 0))
        basis = torch.stack([f00, f10 - f00, f01 - f00, f11 - f10 - f01 + f00], 1)
        p = torch.softmax(raw, 1)

        def back(g):
            gp = g @ basis.t()
            return p * (gp - (p * gp).sum(1, keepdim=True))
        return p @ basis, p @ basis.abs(), back, lambda m: 2 * p * ((m @ basis.abs().t()) + (p * (m @ basis.abs().t())).sum(1, keepdim=True))
    if kind == WALSH:
        m = torch.tensor([[1, -1, -1, 1], [0, 2, 0, -2], [0, 0, 2, -2], [0, 0, 0, 4]], dtype=F64)
        return raw @ m.t(), raw.abs() @ m.abs().t(), lambda g: g @ m, lambda g: g @ m.abs()
    s = torch.sigmoid(raw)
    m = torch.tensor([[1, 0, 0, 0], [-1, 1, 0, 0], [-1, 0, 1, 0], [1, -1, -1, 1]], dtype=F64)
    return s @ m.t(), s @ m.abs().t(), lambda g: (g @ m) * s * (1 - s), lambda g: g @ m.abs()


def layer(x, cand, w, p, kind, inv_tau, gy, pmag=None):
    """``(y, gx, gw, gp)`` of the layer at ``x`` (64 bits), and ``(ymag, gxmag, gwmag, gpmag)``."""
    pmag = p.abs() if pmag is None else pmag
    x, w, p, gy, pmag = (t.detach().cpu().to(F64) for t in (x, w, p, gy, pmag))
    cand = cand.long().cpu()
    got = x[:, cand]

    def evaluate(got, w, p, g, mag):
        a, b = (got * w).sum(-1).unbind(-1)
        z = p[:, 0] + p[:, 1] * a + p[:, 2] * b + p[:, 3] * a * b
        y, gz = z, g
        if kind == WALSH:
            y = torch.sigmoid(z * inv_tau)
            # mag: the sigmoid and its slope are at most 1, off by what z is off
            gz = g * inv_tau * (1 + z * inv_tau) if mag else g * y * (1 - y) * inv_tau
            y = 1 + z * inv_tau if mag else y
        gs = torch.stack([gz * (p[:, 1] + p[:, 3] * b), gz * (p[:, 2] + p[:, 3] * a)], -1)
        if mag and kind == MULTILINEAR:   # (1 - a), (1 - b) and differences of the corners
            gs = gs + 4 * gz.unsqueeze(-1) * (1 + a + b).unsqueeze(-1) * p.sum(1)[:, None]
            y = y + (1 + a) * (1 + b) * p.sum(1)
        gp = torch.stack([gz.sum(0), (gz * a).sum(0), (gz * b).sum(0), (gz * a * b).sum(0)], 1)
        gw = (gs.unsqueeze(-1) * got).sum(0)
        gx = torch.zeros_like(x).index_add_(1, cand.reshape(-1), (gs.unsqueeze(-1) * w).reshape(len(x), -1))
        return y, gx, gw, gp

    return evaluate(got, w, p, gy, False), evaluate(got.abs(), w.abs(), pmag, gy.abs(), True)


def softmax_back(w, gw):
    return w * (gw - (w * gw).sum(-1, keepdim=True))


def softmax_back_mag(w, mag):
    return 2 * w * (mag + (w * mag).sum(-1, keepdim=True))


def close(got, want, bound, what=""):
    """Every value within its bound (and NaN where NaN is wanted)."""
    got, want, bound = got.detach().cpu().to(F64), want.cpu(), bound.cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)}, {tuple(want.shape)} wanted"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    off = (got - want).abs()
    bad = ~torch.isnan(want) & ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} past their bound, the worst "
                           f"{float((off[bad] / bound[bad].clamp_min(1e-300)).max()):.3g} times it")
