"""The operators on logits as a program uses them: networks that learn from a teacher and draw tokens, graphs, streams,
compiled steps, long tensors."""
import pytest
import torch

import logits_oracle as orc
import silogic_amd as sl
from silogic_amd.graphs import CapturedForward

pytestmark = pytest.mark.gpu
DEV = "cuda"
CHECKS = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")


def _student(V=30, L=6, bits=8):
    torch.manual_seed(0)
    enc = sl.TokenEncoder(V, bits, padding_idx=0)
    net = sl.LogicNet(L * bits, 4 * V, 2, num_classes=V, k=4, tau=2.0, seed=0, decoder_ste=False)
    return enc.to(DEV), net.to(DEV)


def test_a_network_learns_from_a_teacher_and_answers():
    """A teacher's logits cut to its largest, a student's step on them, and tokens drawn from the student one after
    another. The step's gradient at the logits is the definition's, and the rest of the network takes it as it takes
    any other; a drawn token is the definition's on the logits that the network gave."""
    enc, net = _student()
    net.train()
    V, N = 30, 50
    ids = torch.randint(0, V, (N, 6), device=DEV)
    values, at = sl.top_logits(3 * torch.randn(N, V, device=DEV), 5)
    labels = at[:, 0].clone()
    labels[3] = -100
    logits = net(enc(ids))
    logits.retain_grad()
    loss = sl.distill_loss(logits, values, at, labels, temperature=2.0)
    loss.backward()
    want = orc.distill(logits.detach(), values, at, labels, 2.0, 0.5, "mean")
    orc.check_distill(loss.detach(), logits.grad, want)
    grads = [p.grad.clone() for p in [*enc.parameters(), *net.parameters()]]
    assert all(torch.isfinite(g).all() for g in grads) and all(g.any() for g in grads)
    for p in [*enc.parameters(), *net.parameters()]:
        p.grad = None
    again = net(enc(ids))
    loss2, g = sl.distill_loss_and_grad(again, values, at, labels, temperature=2.0)
    again.backward(g)
    orc.check_distill(loss2, g, want)
    net.eval()
    window = ids.clone()
    for step in range(5):
        u = torch.rand(N, device=DEV)
        bits = enc.forward_hard(window).float()
        hard = net.sample(bits, u, temperature=0.7, top_k=12, top_p=0.9, min_p=0.01, hard=True)
        counts = net.forward_hard_packed(enc.forward_packed(window), N)
        assert torch.equal(hard.cpu(), orc.sample(counts, u.cpu(), 0.7 * 2.0, 12, 0.9, 0.01))
        soft = net.sample(bits, u, top_p=0.8)
        with torch.no_grad():
            assert torch.equal(soft.cpu(), orc.sample(net(bits), u.cpu(), 1.0, 0, 0.8))
        window = torch.cat([window[:, 1:], hard[:, None]], 1)


def test_a_conv_network_answers():
    torch.manual_seed(0)
    net = sl.LogicTreeNet(2, 8, [4, 8], kernel=3, tree_depth=2, connect="topk", k=4, n_chan=2, num_classes=10, head_widths=[40],
                          residual_init=False).to(DEV).eval()
    x = (torch.rand(20, 2, 8, 8, device=DEV) > 0.5).float()
    u = torch.rand(20, device=DEV)
    t = torch.rand(20, device=DEV) + 0.5
    got = net.sample(x, u, temperature=t, top_k=4, hard=True)
    assert torch.equal(got.cpu(), orc.sample(net.forward_hard(x), u.cpu(), (t * net.head.tau).cpu(), 4))
    assert torch.equal(net.sample(x, u, temperature=0.0, hard=True), net.forward_hard(x).argmax(1))


def test_captured_draws():
    x = torch.randn(33, 6000, device=DEV)
    u = torch.rand(33, device=DEV)
    calls = [lambda x, u: sl.sample_logits(x, u, top_p=0.9), lambda x, u: sl.sample_logits(x, u, top_k=20, min_p=0.01),
             lambda x, u: torch.cat(sl.top_logits(x, 70), 1)]
    steps = [CapturedForward(f, x, u) for f in calls]
    for _ in range(4):
        x.normal_()
        u.uniform_()
        torch.cuda.synchronize()
        for f, step in zip(calls, steps):
            got = step().clone()
            assert torch.equal(got, f(x.clone(), u.clone()))


@pytest.mark.parametrize("N,V", [(40, 500), (4, 50000), (300, 9000)])
def test_captured_training(N, V):
    """Two graphs of different sizes and the eager step in turn: none disturbs another's workspace."""
    def inputs(N, V):
        x = torch.randn(N, V, device=DEV)
        values, ids = sl.top_logits(2 * torch.randn(N, V, device=DEV), 9)
        return [x, values, ids, ids[:, 1].contiguous()]

    def step(x, values, ids, labels):
        s = x.detach().requires_grad_()
        loss = sl.distill_loss(s, values, ids, labels, 2.0)
        return [loss.detach(), torch.autograd.grad(loss, [s])[0], *sl.distill_loss_and_grad(x, values, ids, labels, 2.0, scale=3.0)]

    sets = [inputs(N, V), inputs(N + 3, V + 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            step(*s)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in sets], []
    for graph, s in zip(graphs, sets):
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(*s))
    for _ in range(4):
        for s in sets:
            for old, new in zip(s, inputs(*s[0].shape)):
                old.copy_(new)
        for graph in graphs:
            graph.replay()
        for s, out in zip(sets, outs):
            want = step(*[t.clone() for t in s])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_on_another_stream():
    side = torch.cuda.Stream()
    x, u = torch.randn(64, 20000, device=DEV), torch.rand(64, device=DEV)
    values, ids = sl.top_logits(x, 30)
    want = [sl.sample_logits(x, u, top_p=0.9), *sl.distill_loss_and_grad(x, values, ids)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [sl.sample_logits(x, u, top_p=0.9), *sl.distill_loss_and_grad(x, values, ids)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_and_checked():
    x = torch.randn(9, 50, device=DEV)
    values, ids = sl.top_logits(x, 6)
    labels = ids[:, 2].contiguous()
    s = x.clone().requires_grad_()
    want = sl.distill_loss(s, values, ids, labels, 2.0)
    (gw,) = torch.autograd.grad(want, [s])
    f = torch.compile(lambda s: sl.distill_loss(s, values, ids, labels, 2.0), backend="aot_eager", fullgraph=True)
    got = f(s)
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, [s])[0], gw)
    u, k = torch.rand(9, device=DEV), torch.arange(9, device=DEV)
    g = torch.compile(lambda x, u: (*sl.top_logits(x, 4), sl.sample_logits(x, u, 0.8, k, 0.9, mask=x[0] > -1),
                                    *sl.distill_loss_and_grad(x, values, ids)), backend="aot_eager", fullgraph=True)
    for a, b in zip(g(x, u), (*sl.top_logits(x, 4), sl.sample_logits(x, u, 0.8, k, 0.9, mask=x[0] > -1),
                              *sl.distill_loss_and_grad(x, values, ids))):
        assert torch.equal(a, b)
    ns = torch.ops.silogic_hip
    torch.library.opcheck(ns.top_logits.default, (x, 4), test_utils=CHECKS)
    torch.library.opcheck(ns.sample_logits.default, (x, u, 1.0, 0, 0.9, 0.0, None, k, None, None, x > 0), test_utils=CHECKS)
    torch.library.opcheck(ns.distill_loss_grad.default, (x, values, ids, labels, 2.0, 0.5, 2, 1.0), test_utils=CHECKS)
    torch.library.opcheck(ns.distill_loss.default, (s, values, ids, None, 2.0, 0.5, 0), test_utils=CHECKS)
    with pytest.raises(ValueError):
        ns.distill_loss_bwd(x, values, ids, None, 2.0, 0.5, 0, torch.zeros(9, device=DEV), torch.zeros(9, device=DEV))
    with pytest.raises(ValueError):
        ns.sample_logits(x, u[:4], 1.0, 0, 0.9, 0.0, None, None, None, None, None)


def test_logits_past_32_bit_offsets():
    """2.2e9 logits: rows at both ends as they are by themselves."""
    V, N = 65537, 33000
    x = torch.randn(1, V, device=DEV, dtype=torch.bfloat16).repeat(N, 1)
    x[-1] += torch.randn(V, device=DEV, dtype=torch.bfloat16)
    u = torch.rand(N, device=DEV)
    values, ids = sl.top_logits(x, 3)
    labels = ids[:, 0].contiguous()
    loss, grad = sl.distill_loss_and_grad(x, values, ids, labels, 2.0, reduction="none")
    drawn = sl.sample_logits(x, u, top_p=0.9)
    s = x.detach().requires_grad_()
    (auto,) = torch.autograd.grad(sl.distill_loss(s, values, ids, labels, 2.0, reduction="none").sum(), [s])
    for part in (slice(0, 40), slice(N - 40, N)):
        y = x[part].clone()
        v, i = sl.top_logits(y, 3)
        assert torch.equal(values[part], v) and torch.equal(ids[part], i)
        assert torch.equal(drawn[part], sl.sample_logits(y, u[part], top_p=0.9))
        want = orc.distill(y, v, i, i[:, 0], 2.0, 0.5, "none")
        orc.check_distill(loss[part], grad[part], want)
        orc.check_distill(loss[part], auto[part], want)
