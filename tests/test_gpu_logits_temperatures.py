"""The loss against a teacher over the whole range of temperatures, 1e-4 to 1e4. Far from 1 the soft loss is T^2 times a
divergence of some T^-2, so that its tolerance here does not grow by T^2 but goes by the loss's own parts."""
import math

import pytest
import torch

import logits_oracle as orc
import silogic_amd as sl

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, F64, EPS = math.inf, torch.float64, orc.EPS


def _far(x, values, ids, T):
    """The soft loss of each row in 64 bits, and how far 32 bits may be off, for T over 4.

    Where the entries name more than half of p, the loss over T^2 is sum_j q_j f(r_j) + R with f(r) = e^r - 1 - r, r_j =
    log(p / q) at entry j and R = 1 - sum_j p[i_j]. In units of u = 2^-24: d = (x - m) / T and l = (t - top) / T are off by 3
    of themselves each (a difference, 1 / T, a product), r by one of d - l, of D = log Z - log total and of itself, each; f
    has a slope of |e^r - 1|, so that this counts |p - q|, and its square q; f's own value is off by 32 (at r = 1/2 the
    roundings of e^r, 3.3 of them, and of e^r - 1 over f = 0.149; its series by less). A share q is off by 3 of its l and of
    the mean one, 4 for two exponentials, K / 64 + 7 for its sum's chain and 4 for the quotient and products; the entries'
    terms are added in a chain of K / 64 + 7. An exponential of R is off by 6 of its d and 4: that counts the p of a token
    times how far it is from being named once, 64-bit sums 2^-53 times their chain. What Z and total have in common, their
    exponentials' mean errors, counts R once (the sum over entries takes it by 1 - R) and its square.
    Where they name half or less the loss over T^2 is at least log 2 and its terms, of the sizes of d, l, log Z and log
    total, are off by the same shares of them; Z is a sum of chains of V / 64 + 64 of three roundings each."""
    x, t = x.detach().cpu().to(F64), values.detach().cpu().to(F64) / T
    ids, V, K = ids.cpu(), x.shape[1], ids.shape[1]
    there = (ids >= 0) & (ids < V) & (t != -INF)
    at = torch.where(there, ids, torch.zeros_like(ids))
    t = t.masked_fill(~there, -INF)
    q, lq, lp = torch.softmax(t, 1), torch.log_softmax(t, 1), torch.log_softmax(x / T, 1)
    some = q > 0
    only = lambda v: torch.where(some & v.isfinite(), v, torch.zeros_like(v))  # noqa: E731
    pall = lp.exp()
    dall = (x.amax(1, keepdim=True) - x) / T
    dall = torch.where(dall.isfinite(), dall, torch.zeros_like(dall))
    l, d, p = only(t.amax(1, keepdim=True) - t), only(dall.gather(1, at)), only(pall.gather(1, at))  # noqa: E741
    kl = torch.where(some, q * (lq - lp.gather(1, at)), torch.zeros_like(q)).sum(1)
    logz, logt = -lp.amax(1), -lq.amax(1)                                # of the sums of exp((x - m) / T), exp((t - top) / T)
    named = torch.zeros_like(x).scatter_add_(1, at, some.to(F64))
    rest, parts = (1 - p.sum(1)).abs(), pall * (1 - named).abs()
    lmean, dmean, chain = (q * l).sum(1), (pall * dall).sum(1), K / 64 + 7
    share = (3 * l + 3 * lmean[:, None] + chain + 8) * EPS
    off_r = (3 * (d + l) + 3 * ((d - l).abs() + (logz - logt).abs()[:, None])) * EPS
    common = (6 * dmean + 3 * lmean + 8) * EPS
    near = ((p - q).abs() * off_r + q * off_r ** 2 + q * f(only(lp.gather(1, at) - lq)) * (share + (32 + chain) * EPS)).sum(1) + \
        (parts * (6 * dall + 4) * EPS).sum(1) + (V / 64 + 7) * 2.0 ** -52 + rest * (common + 2 * EPS) + common ** 2
    size = (q * (d + l)).sum(1) + logz + logt
    off = (share.amax(1) + (chain + 12) * EPS) * size + (3 * (V / 64 + 64) + 6 * dmean + 3 * lmean + chain + 8) * EPS
    half = p.sum(1) - 0.5
    tol = torch.where(half.abs() < 1e-4, torch.maximum(near, off), torch.where(half > 0, near, off))
    return T * T * kl, T * T * (tol + 4 * EPS * kl.abs())


def f(r):
    """e^r - 1 - r without cancellation."""
    series = sum(r ** n / math.factorial(n) for n in range(2, 16))
    return torch.where(r.abs() < 0.5, series, torch.expm1(r) - r)


def _check(x, values, ids, T, what):
    x, values, ids = x.to(DEV), values.to(DEV), ids.to(DEV)
    want, tol = _far(x, values, ids, T)
    s = x.clone().requires_grad_()
    loss = sl.distill_loss(s, values, ids, temperature=T, reduction="none")
    orc.close(loss, want, tol, f"{what} T={T}")
    both, grad = sl.distill_loss_and_grad(x, values, ids, temperature=T, reduction="none")
    orc.close(both, want, tol, f"{what} T={T} both")
    assert bool((loss >= 0).all()) and bool((both >= 0).all())
    full = orc.distill(x, values, ids, None, T, 0.5, "none")
    for g in (grad, torch.autograd.grad(loss.sum(), [s])[0]):
        orc.close(g, full["grad"], full["grad_tol"] + (full["grad"].abs() + full["grad_tol"]) * orc.HALF[x.dtype] + orc.TINY[x.dtype], what)
    y = ids[:, 0].clamp(min=0)
    hard = torch.nn.functional.cross_entropy(x.to(F64), y, reduction="none").cpu()
    for reduction in ("mean", "sum"):
        mixed = sl.distill_loss(x, values, ids, y, T, 0.25, reduction)
        one = sl.distill_loss_and_grad(x, values, ids, y, T, 0.25, reduction)[0]
        whole = 0.75 * want + 0.25 * hard
        room = 0.75 * tol + EPS * ((x.shape[1] / 16 + 600) * (hard + 1) + 4 * whole)
        whole, room = (v.mean() if reduction == "mean" else v.sum() for v in (whole, room))
        for v in (mixed, one):
            orc.close(v, whole, room + 4 * EPS * whole.abs(), f"{what} T={T} {reduction}")


def _student(N, V, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = (2.5 * torch.randn(N, V, generator=g)).to(dtype)
    return x, x.float() + torch.randn(N, V, generator=g)


FAR = [4.5, 30.0, 100.0, 1000.0, 1e4]


@pytest.mark.parametrize("T", FAR)
@pytest.mark.parametrize("V,K", [(1, 1), (2, 2), (10, 10), (16, 16), (257, 257), (1000, 1000), (1000, 999), (1000, 600), (1000, 400),
                                 (1024, 1024), (3000, 100)])
def test_far_temperatures(V, K, T):
    """A teacher that names every class, all but one, most, few."""
    for N in (3, 600):
        x, t = _student(N, V, V + K)
        values, ids = torch.topk(t, K, dim=1)
        _check(x, values, ids, T, f"V={V} K={K} N={N}")


@pytest.mark.parametrize("T", FAR)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_far_temperatures_in_16_bits(dtype, T):
    for V in (10, 500):
        x, t = _student(5, V, V, dtype)
        values, ids = torch.topk(t, V, dim=1)
        _check(x, values.to(dtype), ids, T, f"V={V} {dtype}")


@pytest.mark.parametrize("T", FAR)
def test_far_temperatures_of_masked_students(T):
    """Long rows of which only the named tokens have a logit, in parts and one a workgroup; a named one without."""
    for N, V in ((4, 9001), (4, 60000), (520, 5003)):
        x, t = _student(N, V, V)
        values, ids = torch.topk(t, 20, dim=1)
        x = torch.full_like(x, -INF).scatter_(1, ids, x.gather(1, ids))
        _check(x, values, ids, T, f"V={V} masked")
        loss = sl.distill_loss(x.scatter(1, ids[:, :1], -INF).to(DEV), values.to(DEV), ids.to(DEV), temperature=T, reduction="none")
        assert bool((loss == INF).all())


@pytest.mark.parametrize("T", FAR)
def test_far_temperatures_of_wide_logits(T):
    """Logits as far apart as the temperature: neither softmax is flat, and the student is near its teacher."""
    x, t = _student(40, 300, 7)
    values, ids = torch.topk(T * (x + 0.01 * t), 200, dim=1)
    _check(T * x, values, ids, T, "wide")


@pytest.mark.parametrize("T", FAR)
def test_far_temperatures_of_absent_and_repeated_entries(T):
    x, t = _student(6, 30, 9)
    values, ids = torch.topk(t, 30, dim=1)
    ids[0, 3:] = -1
    ids[1, ::2] = 40
    values[2, 5] = -INF
    ids[3, 1] = ids[3, 0]
    ids[4, 5:12] = ids[4, 5]
    values[5, 10:] = -1e30
    want, tol = _far(x, values, ids, T)
    for loss in (sl.distill_loss(x.to(DEV), values.to(DEV), ids.to(DEV), temperature=T, reduction="none"),
                 sl.distill_loss_and_grad(x.to(DEV), values.to(DEV), ids.to(DEV), temperature=T, reduction="none")[0]):
        orc.close(loss, want, tol, f"T={T}")


@pytest.mark.parametrize("T", [1e-4, 1e-3, 1e-2, 0.1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_near_temperatures(T, dtype):
    """Softmaxes of one token: exponents 10^4 times the logits' differences. Against the definition, in the tolerance that
    the other temperatures have."""
    for N, V in ((5, 40), (5, 9001), (600, 300)):
        x, t = _student(N, V, V, dtype)
        values, ids = torch.topk(t, 20, dim=1)
        labels = ids[:, 3].clone()
        labels[1] = -100
        ids[2] = -1
        given = [v.to(DEV) for v in (x, values.to(dtype), ids, labels)]
        s = given[0].clone().requires_grad_()
        loss = sl.distill_loss(s, *given[1:], T, 0.3, "none")
        (g,) = torch.autograd.grad(loss.sum(), [s])
        want = orc.distill(*given, T, 0.3, "none")
        orc.check_distill(loss, g, want, f"T={T}")
        orc.check_distill(*sl.distill_loss_and_grad(*given, T, 0.3, "none"), want, f"T={T} both")
