"""Arguments of the gate layers that keep 8 bits, on the GPU: refused before any launch."""
import pytest
import torch

from silogic_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _args(B=6, IN=9, OUT=5, K=3):
    torch.manual_seed(0)
    return dict(x=torch.rand(B, IN, device=DEV), cand=torch.randint(0, IN, (OUT, 2, K), device=DEV, dtype=torch.int32),
                conn=torch.randn(OUT, 2, K, device=DEV), raw=torch.randn(OUT, 16, device=DEV), node_kind=ops.GATE16)


@pytest.mark.parametrize("grad", [False, True])
def test_layer(grad):
    good = _args()
    good["x"].requires_grad_(grad)
    y = ops.fc_layer8(**good)
    for name in ("cand", "conn", "raw"):
        with pytest.raises(RuntimeError, match="GPU"):
            ops.fc_layer8(**{**good, name: good[name].cpu()})
        with pytest.raises(ValueError):
            ops.fc_layer8(**{**good, name: good[name][:4]})
    assert torch.equal(ops.fc_layer8(**good), y)


def test_backward_operators():
    """The operators that a compiled backward calls, with codes, rows and parameters that do not belong together."""
    a = _args()
    op = torch.ops.silogic_hip
    y, codes, rows, w, kept = op.fc_layer8(a["x"], a["cand"], a["conn"], a["raw"], ops.GATE16, 1.0)
    gy = torch.rand_like(y)

    def layer(codes=codes, rows=rows, w=w, kept=kept, in_dim=9, gy=gy):
        return op.fc_layer8_bwd(codes, rows, a["cand"], w, kept, in_dim, ops.GATE16, 1.0, gy, True, True, True)

    def soft(codes=codes, rows=rows, w=w, npar=kept[:5], in_dim=9, gy=gy):
        return op.fc_soft8_bwd(codes, rows, a["cand"], w, npar, in_dim, ops.GATE16, 1.0, gy, True, True, True)

    gx = layer()[0]
    assert torch.equal(soft()[0], gx)
    spread = torch.zeros((2, 12, 8), device=DEV, dtype=torch.uint8)
    spread[..., ::2] = codes
    assert torch.equal(layer(codes=spread[..., ::2])[0], gx)   # another layout of the same codes
    for call in (layer, soft):
        for bad in (dict(in_dim=100), dict(codes=codes[:1]), dict(rows=rows[:, :1]), dict(w=w[:4]), dict(gy=gy[:5])):
            with pytest.raises(ValueError):
                call(**bad)
    with pytest.raises(ValueError):
        layer(kept=kept[:4])
    with pytest.raises(ValueError):
        layer(kept=kept[:9])
    with pytest.raises(ValueError):
        soft(npar=kept[:4])
