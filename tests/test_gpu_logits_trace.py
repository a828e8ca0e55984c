"""The operators on logits traced on the GPU: the graph gives what the calls give, on new inputs too."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

import silogic_amd as sl

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(N, V, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, V, device=DEV, generator=g)
    values, ids = sl.top_logits(x + torch.randn(N, V, device=DEV, generator=g), 5)
    return x, values, ids, ids[:, 1].contiguous(), torch.rand(N, device=DEV, generator=g)


def _all(x, values, ids, labels, u):
    s = x.detach().requires_grad_()
    loss = sl.distill_loss(s, values, ids, labels, 2.0)
    return [loss.detach(), torch.autograd.grad(loss, [s])[0], *sl.distill_loss_and_grad(x, values, ids, labels, 2.0),
            *sl.top_logits(x, 7), sl.sample_logits(x, u, top_p=0.9), sl.sample_logits(x, u, u + 0.5, top_k=3)]


@pytest.mark.parametrize("tracing", ["real", "symbolic"])
def test_a_traced_step_runs_on_new_inputs(tracing):
    graph = make_fx(_all, tracing_mode=tracing)(*_inputs(9, 50, 1))
    for seed in (1, 2):
        given = _inputs(9, 50, seed)
        for got, want in zip(graph(*given), _all(*given)):
            assert torch.equal(got, want)


def test_a_mode_sees_the_operators():
    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, f, types, args=(), kwargs=None):
            self.names.append(str(f))
            return f(*args, **(kwargs or {}))

    given = _inputs(9, 50, 3)
    want = _all(*given)
    with Seen() as mode:
        got = _all(*given)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for name in ("top_logits", "sample_logits", "distill_loss", "distill_loss_bwd", "distill_loss_grad"):
        assert f"silogic_hip.{name}.default" in mode.names


def test_the_loss_by_functionalized_code():
    given = _inputs(9, 50, 4)
    call = lambda x, v, i, y, u: sl.distill_loss_and_grad(x, v, i, y)[1]  # noqa: E731
    assert torch.equal(torch.func.functionalize(call)(*given), call(*given))


def test_a_recorded_call_runs_on_new_inputs():
    """torch.jit.trace records operators, too."""
    call = lambda x, u: (sl.sample_logits(x, u, top_p=0.9), *sl.top_logits(x, 4))  # noqa: E731
    x, _, _, _, u = _inputs(9, 50, 5)
    recorded = torch.jit.trace(call, (x, u))
    x, _, _, _, u = _inputs(9, 50, 6)
    for got, want in zip(recorded(x, u), call(x, u)):
        assert torch.equal(got, want)
