"""Refusals of the gate layers that keep 8 bits: none of these calls reaches a GPU."""
import pytest
import torch

from silogic_amd import ops


def _args(OUT=5, K=3, kind=ops.GATE16):
    return dict(x=torch.rand(2, 9), cand=torch.zeros((OUT, 2, K), dtype=torch.int32), conn=torch.rand(OUT, 2, K),
                raw=torch.rand(OUT, 16 if kind == ops.GATE16 else 4), node_kind=kind)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("kind", [ops.GATE16, ops.WALSH])
@pytest.mark.parametrize("bad", [dict(conn=torch.rand(5, 2, 2)), dict(conn=torch.rand(4, 2, 3)), dict(conn=torch.rand(5)),
                                 dict(raw=torch.rand(4, 16)), dict(raw=torch.rand(5, 5)), dict(raw=torch.rand(5)),
                                 dict(x=torch.rand(9)), dict(x=torch.rand(2, 0))])
def test_shapes_with_and_without_gradients(grad, kind, bad):
    """The same refusals where nothing is kept: the forward then reads the parameters just as well."""
    args = {**_args(kind=kind), **bad}
    args["x"].requires_grad_(grad)
    with pytest.raises(ValueError, match="8-bit activations"):
        ops.fc_layer8(**args)


@pytest.mark.parametrize("grad", [False, True])
def test_candidates_with_and_without_gradients(grad):
    for cand in (torch.zeros(5, 2, 17), torch.zeros(5, 4, 3), torch.zeros(0, 2, 3)):
        args = _args()
        args["x"].requires_grad_(grad)
        with pytest.raises(NotImplementedError):
            ops.fc_layer8(**{**args, "cand": cand})


@pytest.mark.parametrize("grad", [False, True])
def test_on_the_cpu(grad):
    args = _args()
    args["x"].requires_grad_(grad)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.fc_layer8(**args)
