"""The loss against a teacher at alpha 0 and 1: the term that has no share counts nothing, whatever its values are, in the
loss and in the gradient, by autograd and from one call."""
import math

import pytest
import torch

import logits_oracle as orc
import silogic_amd as sl

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan


def _rows(N, V):
    g = torch.Generator().manual_seed(V)
    x = 2 * torch.randn(N, V, generator=g)
    values, ids = torch.topk(x + torch.randn(N, V, generator=g), 6, dim=1)
    return x, values, ids, torch.randint(0, V, (N,), generator=g)


def _check(x, values, ids, labels, want, T, alpha, reduction):
    x, values, ids, labels = (t.to(DEV) for t in (x, values, ids, labels))
    s = x.clone().requires_grad_()
    loss = sl.distill_loss(s, values, ids, labels, T, alpha, reduction)
    (g,) = torch.autograd.grad(loss.sum(), [s])
    orc.check_distill(loss, g, want, "autograd")
    orc.check_distill(*sl.distill_loss_and_grad(x, values, ids, labels, T, alpha, reduction), want, "one call")


@pytest.mark.parametrize("N,V", [(5, 40), (5, 3000), (4, 20000), (520, 40), (520, 3000), (520, 9000)])
@pytest.mark.parametrize("T", [1.0, 2.0, 3.0, 100.0])
def test_labels_alone(N, V, T):
    x, values, ids, labels = _rows(N, V)
    labels[:4] = (ids[:4, 5] + 1) % V
    for reduction in ("none", "mean"):
        want = orc.distill(x, values, torch.full_like(ids, -1), labels, T, 1.0, reduction)
        _check(x, values, ids, labels, want, T, 1.0, reduction)
        bad = values.clone()
        bad[0, 1], bad[1, 2], bad[2] = NAN, INF, NAN
        _check(x, bad, ids, labels, want, T, 1.0, reduction)
        masked = x.clone()
        masked[3, ids[3, 0]] = -INF     # what the teacher says and the student rules out
        labels[3] = ids[3, 1]
        want = orc.distill(masked, values, torch.full_like(ids, -1), labels, T, 1.0, reduction)
        _check(masked, bad, ids, labels, want, T, 1.0, reduction)


@pytest.mark.parametrize("N,V", [(5, 40), (4, 20000), (520, 3000)])
@pytest.mark.parametrize("T", [1.0, 2.0, 3.0])
def test_the_teacher_alone(N, V, T):
    x, values, ids, labels = _rows(N, V)
    for n in range(3):
        labels[n] = next(i for i in range(V) if i not in ids[n].tolist())
        x[n, labels[n]] = -INF
    for reduction in ("none", "mean"):
        want = orc.distill(x, values, ids, torch.full_like(labels, -100), T, 0.0, reduction)
        _check(x, values, ids, labels, want, T, 0.0, reduction)
