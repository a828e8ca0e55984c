"""Refusals of the gate layers that keep 8 bits: none of these calls reaches a GPU."""
import pytest
import torch

import silogic_amd as sl
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


def _back(B=6, IN=9, OUT=5, K=3):
    return dict(codes=torch.zeros(((B + 3) // 4, (IN + 3) // 4 * 4, 4), dtype=torch.uint8), rows=torch.zeros(B, 2),
                in_dim=IN, cand=torch.zeros((OUT, 2, K), dtype=torch.int32), w=torch.rand(OUT, 2, K),
                npar=torch.rand(OUT, 4), node_kind=ops.GATE16, inv_tau=1.0, gy=torch.rand(B, OUT))


@pytest.mark.parametrize("bad", [dict(in_dim=13), dict(in_dim=8), dict(in_dim=0), dict(rows=torch.zeros(9, 2)),
                                 dict(rows=torch.zeros(6, 1)), dict(rows=torch.zeros(6, 2).double()),
                                 dict(codes=torch.zeros(2, 12, 4)), dict(codes=torch.zeros(2, 9, 4, dtype=torch.uint8)),
                                 dict(codes=torch.zeros(1, 12, 4, dtype=torch.uint8)),
                                 dict(codes=torch.zeros(96, dtype=torch.uint8)), dict(w=torch.rand(4, 2, 3)),
                                 dict(w=torch.rand(5, 2, 2)), dict(npar=torch.rand(4, 4)), dict(npar=torch.rand(5, 3))])
def test_backward_on_codes(bad):
    """Sizes that the kernel would read past: of the codes, of their rows and of the parameters."""
    with pytest.raises(ValueError, match="8-bit activations"):
        ops.fc_soft_bwd8(**{**_back(), **bad})


def test_backward_on_codes_on_the_cpu():
    with pytest.raises(RuntimeError, match="GPU"):
        ops.fc_soft_bwd8(**_back())
    with pytest.raises(NotImplementedError):
        ops.fc_soft_bwd8(**{**_back(), "cand": torch.zeros(5, 2, 17)})


def test_more_candidates_than_the_backwards_take():
    """2^31 of them: the forward says so, not the backward."""
    few = torch.zeros(1, 1, 1, dtype=torch.int32)
    x = torch.rand(2, 9)
    with pytest.raises(NotImplementedError, match="candidates"):
        ops.check_layer8(x, few.expand(1 << 26, 2, 16))
    ops.check_layer8(x, few.expand((1 << 26) - 1, 2, 16))
    layer = sl.LogicLayer(16, 20, k=16)
    assert layer.takes_rows8()
    layer.out_dim = 1 << 26
    assert not layer.takes_rows8()
    with pytest.raises(ValueError):
        sl.save_activations(layer)


@pytest.mark.parametrize("call", ["layer", "soft", "layer backward", "wide backward"])
def test_launched_from_the_tensors_device(monkeypatch, call):
    """Every launch of a call is made with its tensors' device current: without gradients, where nothing is kept,
    and in backwards that unpack wide rows or share the fp32 layers' kernels."""
    here, launches = [7], []

    class Device:
        def __init__(self, d):
            self.d = torch.device(d)

        def __enter__(self):
            self.old, here[0] = here[0], self.d

        def __exit__(self, *exc):
            here[0] = self.old

    class Lib:
        slg_fc_soft_bwd8_workspace = staticmethod(lambda B, IN, OUT, K: -1 if call == "wide backward" else 16)
        slg_fc_soft_bwd_workspace = staticmethod(lambda B, IN, OUT, K: 16)

    monkeypatch.setattr(ops, "require_gpu", lambda *ts: None)
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    monkeypatch.setattr(ops._lib, "lib", lambda: Lib)
    monkeypatch.setattr(ops._lib, "call", lambda name, *args: launches.append((name, here[0])))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", Device)
    a, b = _args(), _back()
    kept = torch.rand(25, 4)
    if call == "layer":
        ops.fc_layer8(**a)
    elif call == "soft":
        ops.fc_soft8(a["x"], a["cand"], b["w"], b["npar"], ops.GATE16)
    elif call == "layer backward":
        ops.fc_layer8_bwd(b["codes"], b["rows"], b["cand"], b["w"], kept, 9, ops.GATE16, 1.0, b["gy"], True, True, True)
    else:
        ops.fc_soft_bwd8(**b)
    assert launches and all(at == torch.device("cpu") for _, at in launches), launches
