"""The operators on logits under tracers, modes and transforms, without a GPU: each call is one operator in what is
traced, never the memory of its result alone, and what an operator cannot be differentiated by is refused."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import silogic_amd as sl

N, V, K = 4, 20, 3

CALLS = {
    "top_logits": lambda x, v, i, y, u: sl.top_logits(x, K),
    "sample_logits": lambda x, v, i, y, u: sl.sample_logits(x, u, top_p=0.9, mask=x[0] > 0),
    "distill_loss": lambda x, v, i, y, u: sl.distill_loss(x, v, i, y),
    "distill_loss_grad": lambda x, v, i, y, u: sl.distill_loss_and_grad(x, v, i, y, 2.0, scale=0.5),
}


def _inputs(device, requires_grad=False):
    return (torch.empty(N, V, device=device, requires_grad=requires_grad), torch.empty(N, K, device=device),
            torch.empty(N, K, dtype=torch.int64, device=device), torch.empty(N, dtype=torch.int64, device=device),
            torch.empty(N, device=device))


def _nodes(graph, name):
    return [n for n in graph.graph.nodes if str(n.target) == f"silogic_hip.{name}.default"]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_a_traced_call_is_its_operator(name, requires_grad):
    with FakeTensorMode():
        graph = make_fx(CALLS[name])(*_inputs("cuda", requires_grad))
    assert len(_nodes(graph, name)) == 1
    assert not [n for n in graph.graph.nodes if "new_empty" in str(n.target)]


def test_results_of_fake_tensors():
    with FakeTensorMode():
        x, v, i, y, u = _inputs("cuda")
        values, ids = sl.top_logits(x.bfloat16().view(2, 2, V), K)
        assert values.shape == ids.shape == (2, 2, K) and values.dtype == torch.bfloat16 and ids.dtype == torch.int64
        token = sl.sample_logits(x.view(2, 2, V), u.view(2, 2), temperature=u.view(2, 2), top_k=2)
        assert token.shape == (2, 2) and token.dtype == torch.int64
        assert sl.distill_loss(x, v, i).shape == () and sl.distill_loss(x, v, i, y, reduction="none").shape == (N,)
        loss, grad = sl.distill_loss_and_grad(x.half(), v, i, reduction="sum")
        assert loss.dtype == torch.float32 and grad.shape == x.shape and grad.dtype == torch.float16
    x = _inputs("cpu")[0]
    with pytest.raises(RuntimeError, match="GPU"):   # not taken for fake ones
        sl.top_logits(x, K)


def test_a_traced_loss_and_its_gradient_are_operators():
    def step(x, v, i, y):
        loss, _ = torch.ops.silogic_hip.distill_loss(x, v, i, y, 2.0, 0.5, 2)
        return torch.autograd.grad(loss, [x])

    graph = make_fx(step)(*_inputs("meta", True)[:4])   # as the call above gives it
    assert len(_nodes(graph, "distill_loss")) == len(_nodes(graph, "distill_loss_bwd")) == 1


@pytest.mark.parametrize("name", CALLS)
def test_transforms_are_refused(name):
    x, u = torch.randn(N, V), torch.rand(N)
    v, i = torch.topk(x, K)
    y = i[:, 0]
    first = lambda r: r[0] if isinstance(r, tuple) else r  # noqa: E731
    call = lambda x: first(CALLS[name](x, v, i, y, u)).sum()  # noqa: E731
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.vmap(lambda x, u, v, i, y: CALLS[name](x[None], v[None], i[None], y[None], u[None]))(x, u, v, i, y)
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.grad(call)(x)
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.jvp(call, (x,), (x,))


@pytest.mark.parametrize("requires_grad", [False, True])
def test_a_tangent_of_the_logits_is_not_lost(requires_grad):
    x = torch.randn(N, V, requires_grad=requires_grad)
    v, i = torch.topk(x.detach(), K)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        sl.distill_loss(forward_ad.make_dual(x, torch.ones(N, V)), v, i)
