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
