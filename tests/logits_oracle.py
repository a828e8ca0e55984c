"""What the operators on logits are in 64 bits, on the CPU, with the error that 32-bit arithmetic may add."""
import math

import torch

F64 = torch.float64
EPS = 2.0 ** -24   # unit rounding of fp32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# exponentials under 2^-126 count 0, times factors of 4 at most; fp16's smallest step
TINY = {torch.float32: 2.0 ** -124, torch.bfloat16: 2.0 ** -124, torch.float16: 2.0 ** -25}


def top(x, k):
    """Values and ids, by value, then by id; -inf and -1 past the tokens that are there."""
    x = x.detach().cpu().to(F64)
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x) + 0.0
    v, i = torch.sort(x, dim=-1, descending=True, stable=True)
    v, i = v[..., :k], i[..., :k]
    return v, torch.where(v > -math.inf, i, torch.full_like(i, -1))


def sample(x, u, t=1.0, k=0, p=1.0, m=0.0, mask=None):
    """Token of each row of x [N, V] by the definition: sorted, cut, summed."""
    x = x.detach().cpu().to(F64)
    N, V = x.shape
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x) + 0.0
    if mask is not None:
        x = x.masked_fill(~mask.cpu().expand(N, V), -math.inf)
    col = lambda v: [float(w) for w in (v.tolist() if torch.is_tensor(v) else [v] * N)]  # noqa: E731
    T, k, p, m, u = (col(v) for v in (t, k, p, m, u.float()))
    out = []
    for n in range(N):
        v, order = torch.sort(x[n], descending=True, stable=True)
        there = int((v > -math.inf).sum())
        if not there:
            out.append(-1)
            continue
        if not T[n] > 0:
            out.append(int(order[0]))
            continue
        v = v[:there]
        if k[n] > 0:
            v = v[:int(min(k[n], there))]
        d = torch.where(v == v[0], torch.zeros_like(v), v - v[0])
        w = torch.exp(d / T[n]).nan_to_num(0.0)   # an infinite temperature under an infinite logit
        run = w.cumsum(0)
        keep = w >= min(max(m[n], 0.0), 1.0) if m[n] > 0 else torch.ones_like(w, dtype=torch.bool)
        if p[n] < 1:
            keep &= run - w < max(p[n], 0.0) * run[-1]
        keep[0] = True
        w = w[keep]
        run = w.cumsum(0)
        target = min(max(u[n], 0.0), 1.0) * float(run[-1]) if u[n] == u[n] else 0.0
        w = (run > target).nonzero()
        out.append(int(order[w[0, 0] if len(w) else (run > float(run[-1]) * (1 - 2 ** -52)).nonzero()[0, 0]]))
    return torch.tensor(out, dtype=torch.int64)


def distill(x, values, ids, labels, T, alpha, reduction, upstream=None):
    """Loss and gradient of rows x [N, V], and how far 32-bit results may be off: {"loss", "loss_tol", "grad",
    "grad_tol"}; the gradient's tolerance without its last rounding.

    p = exp((x - m) c) / Z with u = 2^-24: the difference, the factor c = log2 e / T (three roundings) and the
    product shift the exponent, of size d = (m - x) / T, by at most 6 u d; the exponential is off by 2 u at most, a
    sum of n terms in a chain of at most n / 64 + 64 by three roundings a step (a term, its maximum's change, the
    sum), the quotient and the factors by 8 u. The loss's terms are sums of numbers of sizes d, log Z and those of
    the teacher, each off by a few roundings."""
    x, values = x.detach().cpu().to(F64), values.detach().cpu().to(F64)
    ids = ids.cpu().long()
    N, V = x.shape
    K = values.shape[1]
    there = (ids >= 0) & (ids < V) & (values != -math.inf)
    at = torch.where(there, ids, torch.zeros_like(ids))
    t = torch.where(there, values / T, torch.full_like(values, -math.inf))
    alive = ~(x == -math.inf).all(1)
    given = there.any(1)
    used = given if labels is None else given | ((labels.cpu() >= 0) & (labels.cpu() < V))
    x = torch.where(used[:, None], x, torch.zeros_like(x))   # a row without a term is not looked at
    soft = given & alive
    q = torch.where(there & soft[:, None], torch.softmax(torch.where(given[:, None], t, torch.zeros_like(t)), 1),
                    torch.zeros_like(t))
    whole = torch.zeros(N, V, dtype=F64).scatter_add_(1, at, q)
    xa = torch.where(alive[:, None], x, torch.zeros_like(x))
    lp, lp1 = torch.log_softmax(xa / T, 1), torch.log_softmax(xa, 1)
    share = 1.0 if labels is None else 1.0 - alpha
    a_s = share * soft
    logq = torch.where(q > 0, torch.log(torch.where(q > 0, q, torch.ones_like(q))), torch.zeros_like(q))
    terms = torch.where(q > 0, q * (logq - lp.gather(1, at)), torch.zeros_like(q))
    loss = a_s * T * T * terms.sum(1)
    p = lp.exp() * soft[:, None]
    grad = (a_s * T)[:, None] * (p - whole)
    counts = given
    top = xa.amax(1, keepdim=True)
    d = torch.where(xa > -math.inf, (top - xa), torch.zeros_like(xa))
    relz = (6 * (d * torch.exp(-d / T)).sum(1) / T / torch.exp(-d / T).sum(1) + 3 * (V / 64 + 64) + 16)[:, None] * EPS
    dt = torch.where(there & soft[:, None], t.masked_fill(~there, -math.inf).amax(1, keepdim=True) - t, torch.zeros_like(t))
    relq = (12 * dt.masked_fill(q == 0, 0).amax(1, keepdim=True) + 3 * (K / 64 + 64) + 16) * EPS
    qtol = torch.zeros(N, V, dtype=F64).scatter_add_(1, at, q * (relq + (6 * dt.masked_fill(q == 0, 0) + K) * EPS))
    ptol = p * (relz + (6 * d / T + 10) * EPS)
    grad_tol = (a_s * T)[:, None] * (ptol + qtol)
    big = (torch.where(q > 0, dt, torch.zeros_like(dt)) + torch.where(q > 0, (d / T).gather(1, at), torch.zeros_like(q)) +
           math.log(V) + math.log(K + 1) + 1)
    size = torch.where(q > 0, q * (relq * big + relz + relq + (12 + K / 32) * EPS * big), torch.zeros_like(q))
    loss_tol = a_s * T * T * (size.sum(1) + 8 * EPS * terms.sum(1).abs())
    if labels is not None:
        y = labels.cpu().long()
        known = (y >= 0) & (y < V)
        counts = counts | known
        hard = (known & alive).to(F64) * alpha
        y = torch.where(known, y, torch.zeros_like(y))[:, None]
        loss = loss - torch.where(hard > 0, hard * lp1.gather(1, y)[:, 0], torch.zeros_like(hard))
        one = torch.zeros(N, V, dtype=F64).scatter_(1, y, 1.0)
        grad = grad + hard[:, None] * (lp1.exp() - one)
        relz1 = (6 * (d * torch.exp(-d)).sum(1) / torch.exp(-d).sum(1) + 3 * (V / 64 + 64) + 16)[:, None] * EPS
        grad_tol = grad_tol + hard[:, None] * (lp1.exp() * (relz1 + (6 * d + 10) * EPS) + one * 4 * EPS)
        loss_tol = loss_tol + hard * (relz1[:, 0] + 8 * EPS * (d.gather(1, y)[:, 0] + math.log(V) + 1)) + 4 * EPS * loss.abs()
    n = 1.0
    if reduction == "mean":
        n = max(1, int(counts.sum()))
    g = torch.ones(N, dtype=F64) if upstream is None else upstream.detach().cpu().to(F64).reshape(-1).expand(N)
    grad, grad_tol = grad * (g / n)[:, None], grad_tol * (g.abs() / n)[:, None]
    off = g == 0
    grad[off], grad_tol[off] = 0.0, 0.0
    grad_tol = grad_tol + 6 * EPS * grad.abs()
    if reduction != "none":
        loss, loss_tol = loss.sum() / n, loss_tol.sum() / n + 4 * EPS * loss.abs().sum() / n
    return {"loss": loss, "loss_tol": loss_tol + 2.0 ** -126, "grad": grad, "grad_tol": grad_tol}


def close(got, want, tol, what):
    got = got.detach().cpu().to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(got), (got - want).abs())
    bad = ~same & ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].nan_to_num(math.inf).max()), float(tol.expand_as(off)[bad].max()))


def check_distill(loss, grad, want, what=""):
    close(loss, want["loss"], want["loss_tol"], what + " loss")
    g = want["grad"]
    tol = want["grad_tol"] + (g.abs() + want["grad_tol"]) * HALF[grad.dtype] + TINY[grad.dtype]
    close(grad, g, tol, what + " gradient")
