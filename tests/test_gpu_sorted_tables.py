"""The sort behind the reference tables and the token gradients, by the gradients that run on its order: sizes of
one and several launches, digits of one to three passes, and references that fall on few keys."""
import pytest
import torch

import silogic_amd as sl
from silogic_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64


def _wiring(how, IN, OUT, K, g):
    shape = (OUT, 2, K)
    if how == "uniform":
        return torch.randint(0, IN, shape, generator=g)
    if how == "one":
        return torch.full(shape, IN // 2)
    if how == "ends":
        return torch.randint(0, 2, shape, generator=g) * (IN - 1)
    if how == "window":       # neighbours of the output's place
        at = torch.arange(OUT).view(-1, 1, 1) * IN // OUT
        return (at + torch.randint(-40, 40, shape, generator=g)).clamp(0, IN - 1)
    if how == "low digits":   # keys that differ in their lowest digits alone
        return torch.randint(0, min(IN, 50), shape, generator=g) + max(0, IN // 2 - 50)
    step = max(1, IN // 32)   # "high digits": keys far from each other
    return torch.randint(0, IN // step, shape, generator=g) * step


@pytest.mark.parametrize("how", ["uniform", "one", "ends", "window", "low digits", "high digits"])
@pytest.mark.parametrize("B,IN,OUT,K", [(3, 1500, 257, 8), (3, 1500, 300, 8), (3, 2000, 2000, 8), (2, 4001, 4100, 8), (2, 9000, 2100, 8),
                                        (2, 9000, 2048, 16), (1, 40000, 2100, 4), (2, 16383, 4097, 8), (1, 300000, 3000, 3)])
def test_input_gradient(how, B, IN, OUT, K):
    """An input's gradient is the sum over its references: of whole numbers, so that any order gives the same."""
    g = torch.Generator().manual_seed(0)
    cand = _wiring(how, IN, OUT, K, g)
    w = torch.randint(-2, 3, (OUT, 2, K), generator=g).float()
    gy = torch.randint(-1, 2, (B, OUT), generator=g).float()
    npar = torch.tensor([0.0, 1.0, -1.0, 0.0]).repeat(OUT, 1)   # y = a - b
    x = torch.rand(B, IN, generator=g)
    gx = ops.fc_soft_bwd(*(t.to(DEV) for t in (x, cand.int(), w, npar)), ops.GATE16, 1.0, gy.to(DEV))[0].cpu()
    part = (gy.view(B, OUT, 1, 1) * w * torch.tensor([1.0, -1.0]).view(1, 1, 2, 1)).reshape(B, -1).to(F64)
    want = torch.zeros(B, IN, dtype=F64).index_add_(1, cand.reshape(-1), part)
    assert want.abs().max() < 2 ** 24 and torch.equal(gx.to(F64), want)


@pytest.mark.parametrize("how", ["uniform", "one", "ends", "low digits", "high digits"])
@pytest.mark.parametrize("N,V,D", [(4096, 3000, 3), (4097, 3000, 3), (20000, 1025, 5), (65537, 1500, 4), (131072, 4000, 2),
                                   (131073, 4000, 2), (30000, 70000, 1), (9000, 1200000, 1), (200000, 2000, 2)])
def test_token_gradient(how, N, V, D):
    g = torch.Generator().manual_seed(0)
    ids = _wiring(how, V, N, 1, g)[:, 0, 0]
    gy = torch.randint(-1, 2, (N, D), generator=g).float()
    enc = sl.TokenEncoder.from_weight(torch.zeros(V, D, device=DEV), scale=4.0)   # a slope of 1 at weight 0
    (gt,) = torch.autograd.grad(enc(ids.unsqueeze(1).to(DEV)), [enc.weight], gy.to(DEV))
    want = torch.zeros(V, D, dtype=F64).index_add_(0, ids, gy.to(F64))
    assert torch.equal(gt.cpu().to(F64), want)
