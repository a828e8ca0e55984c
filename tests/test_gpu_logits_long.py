"""The operators on logits where rows are longer than a workgroup's registers, or where many rows take the forms that
few rows do not: against the definitions in 64 bits, on some of the rows."""
import math

import pytest
import torch

import logits_oracle as orc
import silogic_amd as sl

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rows(N, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = 2.5 * torch.randn(N, V, generator=g)
    x[:, :: max(1, V // 9)] += 5 * torch.rand(x[:, :: max(1, V // 9)].shape, generator=g)
    return x.to(dtype)


@pytest.mark.parametrize("V", [33, 257, 1023, 4097, 16385, 33001, 40000, 66001])
@pytest.mark.parametrize("dtype", TYPES)
def test_loss_and_gradient_of_many_rows(V, dtype):
    """A workgroup for each row, with every number of softmaxes; a row without a teacher, without a label, with
    neither, of -inf alone, and with a token named twice."""
    N, K = 515, min(V, 40)
    some = _rows(13, V, dtype, V)
    x = some[torch.arange(N) % 13]
    values, ids = torch.topk(some.float() + torch.randn(13, V, generator=torch.Generator().manual_seed(1)), K, dim=1)
    labels = ids[:, 0].clone()
    ids[1], labels[2] = -1, -100
    ids[3], labels[3] = V, V + 7
    ids[4, 1] = ids[4, 0]
    ids[5, K // 2:] = -5
    x[6::13] = -INF
    pick = torch.arange(N) % 13
    values, ids, labels = values.to(dtype)[pick], ids[pick], labels[pick]
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    at = torch.cat([torch.arange(13), torch.arange(N - 13, N)])
    for lab, T, alpha in ((labels, 2.0, 0.3), (labels, 3.0, 0.3), (labels, 1.0, 0.3), (None, 2.0, 0.3), (labels, 2.0, 0.0), (labels, 1.5, 1.0)):
        loss, grad = sl.distill_loss_and_grad(d(x), d(values), d(ids), d(lab), T, alpha, "none", scale=0.7)
        want = orc.distill(x[at], values[at], ids[at], None if lab is None else lab[at], T, alpha, "none", torch.full((26,), 0.7).float())
        orc.check_distill(loss[at], grad[at], want, f"V={V} {dtype} T={T} alpha={alpha}")
        s = d(x).requires_grad_()
        auto = sl.distill_loss(s, d(values), d(ids), d(lab), T, alpha, "none")
        (g,) = torch.autograd.grad(auto, [s], torch.full((N,), 0.7, device=DEV))
        orc.check_distill(auto[at], g[at], want, f"autograd V={V} {dtype} T={T} alpha={alpha}")
        # the mean over the rows that count: one in 13 has neither
        mean, g = sl.distill_loss_and_grad(d(x), d(values), d(ids), d(lab), T, alpha, "mean")
        there = ((ids >= 0) & (ids < V)).any(1)
        if lab is not None:
            there |= (lab >= 0) & (lab < V)
        n = int(there.sum())
        assert abs(float(mean) - float(loss.double().sum()) / n) <= 4 * orc.EPS * abs(float(loss.double().abs().sum()) / n)
        # a named token's gradient is a difference: its roundings go by the two sides, as the definition's tolerance has it
        part = orc.distill(x[at], values[at], ids[at], None if lab is None else lab[at], T, alpha, "none",
                           torch.full((26,), 1.0 / n, dtype=orc.F64))
        orc.check_distill(loss[at], g[at], part, f"mean V={V} {dtype} T={T} alpha={alpha}")


LIMITS = [dict(), dict(k=40), dict(k=900, t=0.7), dict(p=0.9), dict(p=0.5, t=1.5), dict(m=0.05), dict(p=0.9, m=0.02), dict(k=30, p=0.9), dict(t=0.0),
          dict(t=40.0), dict(t=INF)]


def _check_sample(x, mask=None):
    u = torch.rand(len(x), generator=torch.Generator().manual_seed(5))
    names = dict(t="temperature", k="top_k", p="top_p", m="min_p")
    for limits in LIMITS:
        got = sl.sample_logits(x.to(DEV), u.to(DEV), mask=None if mask is None else mask.to(DEV), **{names[n]: v for n, v in limits.items()})
        assert torch.equal(got.cpu(), orc.sample(x, u, mask=mask, **limits)), limits


@pytest.mark.parametrize("V", [16383, 16388, 32771, 40000, 70003])
@pytest.mark.parametrize("dtype", TYPES)
def test_draws_from_long_rows(V, dtype):
    x = _rows(6, V, dtype, V)
    _check_sample(x)
    mask = torch.rand(6, V, generator=torch.Generator().manual_seed(2)) < 0.4
    mask[0] = False
    mask[1] = False
    mask[1, V - 2] = True
    x[2, ~mask[2]] = NAN
    _check_sample(x, mask)
    x[3, V - 5:] = INF
    x[4] = -INF
    x[4, [7, V - 1]] = 1.5
    x[5, ::2] = -INF
    _check_sample(x)


@pytest.mark.parametrize("V", [16383, 32771, 70003])
@pytest.mark.parametrize("dtype", TYPES)
def test_largest_of_long_rows(V, dtype):
    x = _rows(5, V, dtype, V)
    x[1] = x[1, 0]
    x[2, 9:] = NAN
    x[3, V - 300:] = INF
    for k in (1, 100, 161, 1024):
        values, ids = sl.top_logits(x.to(DEV), k)
        v, i = orc.top(x, k)
        assert torch.equal(ids.cpu(), i) and torch.equal(values.cpu().to(orc.F64), v)


def test_rows_of_odd_strides_and_offsets():
    """Rows that begin anywhere in their memory: groups of 16 bytes are read from any element on."""
    wide = torch.randn(9, 5011, generator=torch.Generator().manual_seed(3))
    for dtype in TYPES:
        y = wide.to(dtype).to(DEV)
        for a in range(9):
            v = y[:, a:a + 5000]
            u = torch.rand(9, device=DEV)
            dense = v.contiguous()
            assert torch.equal(sl.sample_logits(v, u, top_p=0.9), sl.sample_logits(dense, u, top_p=0.9))
            assert torch.equal(sl.top_logits(v, 20)[1], sl.top_logits(dense, 20)[1])
            values, ids = sl.top_logits(dense.flip(0), 20)
            for p, q in zip(sl.distill_loss_and_grad(v, values, ids), sl.distill_loss_and_grad(dense, values, ids)):
                assert torch.equal(p, q)
