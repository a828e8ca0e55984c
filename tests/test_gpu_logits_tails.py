"""Draws from the longest rows: tails of masses far under the largest, which hold little each and much together. Against
sums in 64 bits, to 2^-27 of a row's sum, which is under the steps of a random number near 1."""
import math

import pytest
import torch

import silogic_amd as sl

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64
OFF = 2.0 ** -27 + 2.0 ** -43


def _sums(x, T=1.0, keep=None):
    """Order of a row's tokens, their masses (0 where they are not among the first `keep`) and running sums, in 64 bits."""
    v, order = torch.sort(x.to(F64), descending=True, stable=True)
    w = torch.exp((v - v[0]) / T)
    if keep is not None:
        w[keep:] = 0
    return order, w, w.cumsum(0)


def _check(token, u, order, w, run, total=None):
    """u's place lies in the token's part of the kept sum."""
    total = float(run[-1]) if total is None else total
    at = int((order == int(token)).nonzero()[0, 0])
    off = OFF * float(run[-1])
    want = float(u) * total
    assert w[at] > 0 and run[at] - w[at] - off <= want <= run[at] + off, (int(token), float(u), at)


@pytest.mark.parametrize("V", [(1 << 18) - 1, 1 << 18, 1 << 20, 1 << 24])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_flat_tail_is_drawn(V, dtype):
    """One token and a tail of 3e-12 of its mass each: random numbers up to the last one before 1."""
    x = torch.full((V,), -26.4, device=DEV, dtype=dtype)
    x[7] = 0.0
    order, w, run = _sums(x)
    share = 1.0 - 1.0 / float(run[-1])   # of the tail
    us = [0.0, 0.5, 1.0 - 2.0 * share, 1.0 - 2.0 ** -24] + [1.0 - share * f for f in (0.99, 0.7, 0.5, 0.3, 0.05)]
    u = torch.tensor(us, dtype=torch.float32, device=DEV).clamp(max=1.0 - 2.0 ** -24)
    rows = x.expand(len(us), V)
    got = sl.sample_logits(rows, u)
    assert torch.equal(got, sl.sample_logits(rows.contiguous(), u))
    for token, r in zip(got.tolist(), u.tolist()):
        _check(token, r, order, w, run)
    if share > 2.0 ** -20:
        assert len(set(got.tolist())) > 4
    # the same by limits that keep all of the tail, part of it, or none
    for token, r in zip(sl.sample_logits(rows, u, min_p=1e-12).tolist(), u.tolist()):
        _check(token, r, order, w, run)
    assert sl.sample_logits(rows, u, min_p=1e-11).tolist() == [7] * len(us)
    k = V // 2
    first = _sums(x, keep=k)
    for token, r in zip(sl.sample_logits(rows, u, top_k=k).tolist(), u.tolist()):
        _check(token, r, *first)
    p = 1.0 - 0.4 * share
    total = float(run[int((run - w < p * run[-1]).nonzero()[-1, 0])])
    for token, r in zip(sl.sample_logits(rows, u, top_p=p).tolist(), u.tolist()):
        _check(token, r, order, w, run, total)


@pytest.mark.parametrize("V", [(1 << 18) + 3, 1000003])
@pytest.mark.parametrize("T", [0.3, 1.0, 8.0, math.inf])
def test_long_rows_by_their_sums(V, T):
    """Sums from 1 to V of the largest mass, with masked tokens and infinite ones."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = 4 * torch.randn(6, V, device=DEV, generator=g)
    x[1] = 2.5
    x[2, 5:] = -math.inf
    x[3] -= 30
    x[3, V // 2] = 9
    x[4, ::2] = math.nan
    u = torch.rand(6, device=DEV, generator=g)
    mask = torch.rand(6, V, device=DEV, generator=g) < 0.5
    mask[:, 0] = True
    for m in (None, mask):
        got = sl.sample_logits(x, u, temperature=T, mask=m).tolist()
        for n in range(6):
            y = x[n].nan_to_num(nan=-math.inf, neginf=-math.inf)
            if m is not None:
                y = y.masked_fill(~m[n], -math.inf)
            order, w, run = _sums(y, T)
            w = torch.where(y[order] > -math.inf, w.nan_to_num(0.0), torch.zeros_like(w))   # -inf over an infinite T
            _check(got[n], u[n], order, w, w.cumsum(0))
    x[5, V - 9:] = math.inf
    assert int(sl.sample_logits(x, u, temperature=T)[5]) == V - 9 + int(float(u[5]) * 9)
