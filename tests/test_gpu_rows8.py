"""Activations in 8 bits, the gate layers that keep them for their backward, and the networks that train
on them, against 64-bit oracles."""
import pytest
import torch

import silogic_amd as sl
from silogic_amd import ops
import rows8_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = {"gate16": orc.GATE16, "walsh": orc.WALSH, "multilinear": orc.MULTILINEAR}


def _rows(B, D):
    """Rows of several kinds: soft values of one range each, bits, constants, negative and far offsets."""
    x = torch.rand(B, D)
    for b in range(B):
        if b % 5 == 1:
            x[b] = (x[b] > 0.5).float()
        elif b % 5 == 2:
            x[b] = x[b] * 1e-3 + 0.5
        elif b % 5 == 3:
            x[b] = x[b] * 40 - 30
        elif b % 5 == 4 and b % 2:
            x[b] = 0.25
    return x


@pytest.mark.parametrize("B,D", [(1, 1), (1, 2), (3, 5), (4, 64), (5, 255), (7, 257), (6, 1000), (9, 1025),
                                 (3, 4097), (2, 8193), (5, 16384), (3, 16387), (2, 70001), (70, 33),
                                 (5, 3), (9, 4), (6, 256), (3, 512), (4, 513), (6, 1024), (3, 2048), (5, 2049), (2, 4096),
                                 (3, 8192), (2, 16381), (1, 16383), (5, 16385), (3, 24576), (6, 24577), (9, 32771), (4, 40959),
                                 (7, 40961)])
def test_pack_and_unpack(B, D):
    x = _rows(B, D)
    codes, rows = sl.pack_rows8(x.to(DEV))
    q, lo, step = orc.codes_of(x)
    assert codes.shape == ((B + 3) // 4, D, 4) and rows.shape == (B, 2)
    flat = codes.permute(0, 2, 1).reshape(-1, D).cpu()
    assert torch.equal(flat[:B].float(), q), "codes"
    assert not flat[B:].any(), "codes past the batch"
    assert torch.equal(rows.cpu(), torch.stack([lo, step], 1)), "offsets and steps"
    got = sl.unpack_rows8(codes, rows)
    want = orc.values_of(x)
    orc.close(got, want, orc.EPS * (want.abs() + lo.to(orc.F64).abs()[:, None]), "values")
    # half a step of the exact quantiser, and two roundings of lo and the step's product
    span = (x.amax(1) - x.amin(1)).to(orc.F64)[:, None]
    orc.close(got, x.to(orc.F64), span / 510 + 4 * orc.EPS * (x.abs().to(orc.F64) + span), "values")


def test_bits_come_back_exactly():
    x = (torch.rand(13, 77) > 0.5).float()
    x[3], x[4] = 0.0, 1.0
    assert torch.equal(sl.unpack_rows8(*sl.pack_rows8(x.to(DEV))).cpu(), x)


def test_rows_that_are_not_finite_come_back_as_nan():
    x = torch.rand(6, 40)
    x[0, 3], x[1, 0], x[2, 39] = float("nan"), float("inf"), -float("inf")
    x[3] = torch.linspace(-3e38, 3e38, 40)   # the span overflows
    x[4] = torch.linspace(0, 1e-37, 40)      # 255 / span overflows: all codes 0
    got = sl.unpack_rows8(*sl.pack_rows8(x.to(DEV))).cpu()
    assert torch.isnan(got[:4]).all()
    assert torch.equal(got[4], x[4, :1].expand(40))
    orc.close(got[5:], orc.values_of(x[5:]), 2 * orc.EPS * torch.ones(1, 40))


def test_pack_takes_views_and_other_types():
    x = torch.rand(10, 31, device=DEV)
    for v in (x.t(), x[1:, 3:], x[::2], x.half(), x.bfloat16(), x.double()):
        a, b = sl.pack_rows8(v), sl.pack_rows8(v.float().contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    codes, rows = sl.pack_rows8(x)
    want = sl.unpack_rows8(codes, rows)
    assert torch.equal(sl.unpack_rows8(codes.contiguous(), rows), want)   # another layout of the codes
    assert torch.equal(sl.unpack_rows8(codes[:, :7], rows), want[:, :7])
    assert sl.unpack_rows8(*sl.pack_rows8(x[:0])).shape == (0, 31)


def _problem(kind, B, IN, OUT, K, seed=0, x=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(B, IN, generator=g) if x is None else x
    cand = torch.randint(0, IN, (OUT, 2, K), generator=g, dtype=torch.int32)
    if K > 1 and OUT > 1:
        cand[0] = 0            # one input for every candidate of both operands
        cand[1] = IN - 1
    conn = torch.randn(OUT, 2, K, generator=g)
    raw = torch.randn(OUT, 16 if kind == orc.GATE16 else 4, generator=g)
    gy = torch.randn(B, OUT, generator=g)
    return x, cand, conn, raw, gy


def _grads(x, cand, conn, raw, gy, kind, inv_tau, fn=None):
    leaves = [None if t is None else t.to(DEV).requires_grad_() for t in (x, conn, raw)]
    y = (fn or ops.fc_layer8)(leaves[0], cand.to(DEV), leaves[1], leaves[2], kind, inv_tau)
    inputs = [t for t in leaves if t is not None]
    return (y, *torch.autograd.grad(y, inputs, gy.to(DEV)))


def _check_layer(kind, B, IN, OUT, K, inv_tau, x=None, fn=None):
    x, cand, conn, raw, gy = _problem(kind, B, IN, OUT, K, x=x)
    y, gx, gconn, graw = _grads(x, cand, conn, raw, gy, kind, inv_tau, fn)
    w = torch.softmax(conn.to(orc.F64), -1)
    p, pmag, back, back_mag = orc.poly(kind, raw)
    (yw, *_), (ym, *_) = orc.layer(x, cand, w, p, kind, inv_tau, gy, pmag)
    (_, gxw, gww, gpw), (_, gxm, gwm, gpm) = orc.layer(orc.values_of(x), cand, w, p, kind, inv_tau, gy, pmag)
    # roundings on a path: the softmaxes (K + 6 and 26), the operand (a product, K sums, offset and step: K +
    # 4), the node (12, twice where its slope reads the operands again), then the sums: over the batch for
    # parameters, over an input's references (at most all 2 K OUT) for the input
    n = 4 * K + 80
    orc.close(y, yw, n * orc.EPS * ym, "y")
    refs = torch.bincount(cand.long().reshape(-1), minlength=IN).to(orc.F64)
    orc.close(gx, gxw, (n + refs) * orc.EPS * gxm, "gx")
    n += B
    orc.close(gconn, orc.softmax_back(w, gww), (n + K) * orc.EPS * orc.softmax_back_mag(w, gwm), "gconn")
    orc.close(graw, back(gpw), (n + 20) * orc.EPS * back_mag(gpm), "graw")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("B,IN,OUT,K", [(1, 1, 1, 1), (1, 2, 3, 2), (2, 5, 64, 3), (3, 7, 65, 4), (4, 100, 511, 8),
                                        (5, 131, 513, 5), (63, 64, 1023, 8), (65, 997, 1025, 4),
                                        (130, 300, 77, 16), (33, 2001, 130, 8), (257, 50, 40, 11)])
def test_layer(kind, B, IN, OUT, K):
    _check_layer(KINDS[kind], B, IN, OUT, K, 0.5 if kind == "walsh" else 1.0)


@pytest.mark.parametrize("B,IN,OUT,K", [(1, 2, 169, 11), (5, 1, 900, 16), (3, 3, 5000, 8)])
def test_few_inputs_under_many_outputs(B, IN, OUT, K):
    """Lists of hundreds to tens of thousands of references to one input."""
    _check_layer(orc.MULTILINEAR, B, IN, OUT, K, 1.0)


@pytest.mark.parametrize("IN", [16400, 40960, 40964, 66000])
def test_wide_rows(IN):
    """Rows up to the LDS's 40960 words on the codes, wider ones unpacked."""
    _check_layer(orc.GATE16, 6, IN, 150, 8, 1.0)


@pytest.mark.parametrize("B,IN,OUT,K", [(1, 1, 1, 1), (5, 64, 70, 8), (9, 1280, 700, 4), (130, 1281, 40, 8),
                                        (4100, 1300, 64, 4), (4099, 4099, 65, 3), (33, 10000, 129, 8),
                                        (7, 10177, 30, 8), (6, 16380, 200, 4), (5, 30001, 40, 2), (3, 41000, 50, 8),
                                        (130, 40, 70001, 8), (70, 16400, 60007, 8), (41, 30001, 60001, 8)])
def test_forward_writes_what_pack_writes(B, IN, OUT, K):
    """The codes that a layer's forward makes from its staged tiles (4 and 8 samples, several output chunks a
    tile) or beside them (narrower tiles), and its output, are those of the separate calls; also where the
    layer reads its parameters from records."""
    assert (ops._lib.lib().slg_fc_layer8_fwd_workspace(B, IN, OUT, K) > 0) == (OUT > 60000)
    x, cand, conn, raw, _ = _problem(orc.GATE16, B, IN, OUT, K, x=_rows(B, IN))
    if B > 2:
        x[2, IN // 2] = float("nan")
    x, cand, conn, raw = (t.to(DEV) for t in (x, cand, conn, raw))
    y, codes, rows, w, kept = ops.fc_layer8_fwd(x, cand, conn, raw, orc.GATE16, 1.0)
    want = ops.rows8_pack(x)
    assert torch.equal(codes, want[0]) and torch.equal(rows.isnan(), want[1].isnan())
    assert torch.equal(rows.nan_to_num(7.0), want[1].nan_to_num(7.0))
    yw = ops._fc_soft_launch(x, cand, w, kept[:OUT], orc.GATE16, 1.0)
    assert torch.equal(y.nan_to_num(7.0), yw.nan_to_num(7.0))


@pytest.mark.parametrize("kind", list(KINDS))
def test_layer_of_rows_with_ranges_of_their_own(kind):
    x = _rows(37, 90)
    _check_layer(KINDS[kind], 37, 90, 70, 4, 1.0, x=x)


def test_layer_on_weights_and_node_parameters():
    """fc_soft8, the form of selections that have no kernel of their own."""
    x, cand, conn, raw, gy = _problem(orc.WALSH, 21, 40, 70, 6)
    w, p = torch.softmax(conn, -1), torch.randn(70, 4)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, p)]
    y = ops.fc_soft8(leaves[0], cand.to(DEV), leaves[1], leaves[2], orc.WALSH, 0.7)
    gx, gw, gp = torch.autograd.grad(y, leaves, gy.to(DEV))
    (yw, *_), (ym, *_) = orc.layer(x, cand, w, p, orc.WALSH, 0.7, gy)
    (_, gxw, gww, gpw), (_, gxm, gwm, gpm) = orc.layer(orc.values_of(x), cand, w, p, orc.WALSH, 0.7, gy)
    n = (4 * 6 + 80 + 21 + 20) * orc.EPS
    for got, want, mag in ((y, yw, ym), (gx, gxw, gxm), (gw, gww, gwm), (gp, gpw, gpm)):
        orc.close(got, want, n * mag)


def test_gradient_against_differences():
    """The gradient of the layer at the 8-bit values, by central differences of its 64-bit value there."""
    kind = orc.GATE16
    x, cand, conn, raw, gy = _problem(kind, 9, 12, 8, 3)
    _, gx, gconn, graw = _grads(x, cand, conn, raw, gy, kind, 1.0)
    at = [orc.values_of(x), conn.to(orc.F64), raw.to(orc.F64)]

    def loss(xv, cv, rv):
        p = orc.poly(kind, rv)[0]
        return float((orc.layer(xv, cand, torch.softmax(cv, -1), p, kind, 1.0, gy)[0][0] * gy).sum())

    h = 1e-5
    for k, got in ((0, gx), (1, gconn), (2, graw)):
        for i in range(0, at[k].numel(), 7):
            lo, hi = [t.clone() for t in at], [t.clone() for t in at]
            lo[k].view(-1)[i] -= h
            hi[k].view(-1)[i] += h
            want = (loss(*hi) - loss(*lo)) / (2 * h)
            # h^2 of the third derivative, and fp32's roundings of sums of at most 72 terms of size 1
            assert abs(want - float(got.reshape(-1)[i])) < 1e-8 + 200 * orc.EPS * (1 + abs(want))


def test_only_the_wanted_gradients():
    x, cand, conn, raw, gy = _problem(orc.MULTILINEAR, 18, 33, 65, 4)
    full = _grads(x, cand, conn, raw, gy, orc.MULTILINEAR, 1.0)[1:]
    for k in range(3):
        leaves = [t.to(DEV).requires_grad_(i == k) for i, t in enumerate((x, conn, raw))]
        y = ops.fc_layer8(leaves[0], cand.to(DEV), leaves[1], leaves[2], orc.MULTILINEAR)
        (g,) = torch.autograd.grad(y, [leaves[k]], gy.to(DEV))
        assert torch.equal(g, full[k])


def test_fixed_wiring_and_no_gradient():
    x, cand, _, raw, gy = _problem(orc.GATE16, 10, 20, 30, 1)
    y, gx, graw = _grads(x, cand, None, raw, gy, orc.GATE16, 1.0)
    yr, gxr = _grads(x, cand, torch.zeros(30, 2, 1), raw, gy, orc.GATE16, 1.0)[:2]   # a softmax of one
    assert torch.equal(y, yr) and torch.equal(gx, gxr)
    with torch.no_grad():
        again = ops.fc_layer8(x.to(DEV), cand.to(DEV), None, raw.to(DEV), orc.GATE16)
    # evaluated on the other parameter kernel: same formula, other order of the 16 terms
    assert (again - y).abs().max() < 64 * orc.EPS


def test_empty_batch():
    x, cand, conn, raw, gy = _problem(orc.GATE16, 0, 20, 30, 4)
    y, gx, gconn, graw = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)
    assert y.shape == (0, 30) and gx.shape == (0, 20)
    assert not gconn.any() and not graw.any()


def test_a_row_that_is_not_finite():
    """It reaches the gradients as NaN; the other samples' input gradients are as without it."""
    x, cand, conn, raw, gy = _problem(orc.GATE16, 9, 20, 30, 4)
    clean = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)[1]
    x[5, 7] = float("inf")
    _, gx, gconn, _ = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)
    keep = [b for b in range(9) if b != 5]
    assert torch.equal(gx[keep], clean[keep])
    assert torch.isnan(gconn).any()


def test_the_same_bits_on_every_call_and_on_another_stream():
    x, cand, conn, raw, gy = _problem(orc.GATE16, 300, 500, 700, 8)
    first = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_parameters_may_change_before_the_backward():
    x, cand, conn, raw, gy = _problem(orc.GATE16, 12, 20, 30, 4)
    want = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)
    leaves = [t.to(DEV).requires_grad_() for t in (x, conn, raw)]
    y = ops.fc_layer8(leaves[0], cand.to(DEV), leaves[1], leaves[2], orc.GATE16)
    with torch.no_grad():
        for t in leaves:
            t.mul_(3)
    for a, b in zip(want[1:], torch.autograd.grad(y, leaves, gy.to(DEV))):
        assert torch.equal(a, b)


def test_strides_and_types_of_the_arguments():
    x, cand, conn, raw, gy = _problem(orc.GATE16, 12, 20, 30, 4)
    want = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)
    xt = x.t().contiguous().to(DEV).t().requires_grad_()
    c = torch.cat([conn, conn], -1).to(DEV)[..., :4].requires_grad_()
    r = raw.to(DEV).requires_grad_()
    y = ops.fc_layer8(xt, cand.long().to(DEV), c, r, orc.GATE16)
    g = torch.cat([gy, gy], 1).to(DEV)[:, :30]
    for a, b in zip(want, (y, *torch.autograd.grad(y, [xt, c, r], g))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("node", list(KINDS))
def test_network_keeps_bytes_and_its_outputs(node):
    """A network's outputs stay the same bits, its saved inputs are codes, its gradients the layers' own."""
    torch.manual_seed(0)
    kw = dict(node=node, tau=2.0) if node == "walsh" else dict(node=node)
    net = torch.nn.Sequential(sl.LogicLayer(50, 60, k=4, seed=1, **kw), sl.LogicLayer(60, 40, k=4, seed=2, **kw)).to(DEV)
    x = torch.rand(30, 50, device=DEV)
    gy = torch.randn(30, 40, device=DEV)
    y32 = net(x)
    g32 = torch.autograd.grad(y32, list(net.parameters()), gy)
    assert sl.save_activations(net) == 2
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        y8 = net(x)
    assert torch.equal(y8, y32)
    assert not any(t.dtype == torch.float32 and t.shape[0] == 30 and t.numel() > 60 for t in saved), "an fp32 input is kept"
    # codes of whole tiles and quads, an offset and a step a sample, weights and node parameters
    kept = 5 if node == "gate16" else 1
    assert sum(t.numel() for t in saved if t.dtype == torch.uint8) == sum(
        8 * 4 * ld + 8 * 30 + 8 * out * 4 + 16 * out * kept for ld, out in ((52, 60), (60, 40)))
    for a, b in zip(torch.autograd.grad(y8, list(net.parameters()), gy), g32):
        # inputs off by at most span / 510, twice through softmaxes' slopes: a hundredth of the norm
        assert (a - b).norm() < 0.01 * b.norm() + 1e-6
    assert sl.save_activations(net, 32) == 2
    for a, b in zip(torch.autograd.grad(net(x), list(net.parameters()), gy), g32):
        assert torch.equal(a, b)


def test_gumbel_selections_keep_bytes():
    torch.manual_seed(0)
    for kw in (dict(node="gate16", gate_select="gumbel"), dict(node="walsh", gate_select="gumbel"),
               dict(node="gate16", gate_select="hard")):
        layer = sl.LogicLayer(30, 40, k=4, seed=1, **kw).to(DEV).train()
        sl.save_activations(layer)
        saved = []
        x = torch.rand(10, 30, device=DEV, requires_grad=True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
            y = layer(x)
        assert any(t.dtype == torch.uint8 for t in saved)
        assert not any(t.shape == x.shape and t.dtype == torch.float32 for t in saved)
        torch.manual_seed(3)
        a = torch.autograd.grad(layer(x).sum(), x)[0]
        sl.save_activations(layer, 32)
        torch.manual_seed(3)
        b = torch.autograd.grad(layer(x).sum(), x)[0]
        assert (a - b).norm() < 0.05 * b.norm()


def test_captured_training_step():
    """Forward and backward of a layer in a graph, replayed between eager work on new inputs."""
    x, cand, conn, raw, gy = _problem(orc.GATE16, 40, 60, 70, 8)
    cand = cand.to(DEV)
    sx, sc, sr, sg = (t.to(DEV) for t in (x, conn, raw, gy))

    def step(x, conn, raw, gy):
        leaves = [t.detach().requires_grad_() for t in (x, conn, raw)]
        y = ops.fc_layer8(leaves[0], cand, leaves[1], leaves[2], orc.GATE16)
        return (y, *torch.autograd.grad(y, leaves, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, sc, sr, sg)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):   # two graphs, each with its workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(sx, sc, sr, sg)
        graphs.append((g, out))
    for k in range(4):
        new = [torch.rand_like(t) for t in (sx, sc, sr, sg)]
        for dst, src in zip((sx, sc, sr, sg), new):
            dst.copy_(src)
        for g, _ in graphs:
            g.replay()
        want = step(*new)
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b), f"replay {k}"


def test_compiled_layer():
    layer = sl.LogicLayer(30, 40, k=4, seed=1).to(DEV)
    sl.save_activations(layer)
    x = torch.rand(10, 30, device=DEV)
    y = layer(x)
    want = torch.autograd.grad(y.sum(), list(layer.parameters()))
    c = torch.compile(layer, backend="aot_eager", fullgraph=True)(x)
    assert torch.equal(c, y)
    for a, b in zip(torch.autograd.grad(c.sum(), list(layer.parameters())), want):
        assert torch.equal(a, b)


def test_custom_ops_check():
    x, cand, conn, raw, _ = _problem(orc.GATE16, 6, 9, 8, 3)
    args = [t.to(DEV).requires_grad_() for t in (x, conn, raw)]
    torch.library.opcheck(torch.ops.silogic_hip.fc_layer8, (args[0], cand.to(DEV), args[1], args[2], orc.GATE16, 1.0))
    w, p = torch.softmax(conn, -1).to(DEV).requires_grad_(), torch.rand(8, 4, device=DEV, requires_grad=True)
    torch.library.opcheck(torch.ops.silogic_hip.fc_soft8, (args[0], cand.to(DEV), w, p, orc.WALSH, 0.5))


def test_under_autocast():
    layer = sl.LogicLayer(30, 40, k=4, seed=1).to(DEV)
    sl.save_activations(layer)
    x = torch.rand(10, 30, device=DEV)
    y = layer(x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(layer(x), y)


def test_no_second_derivative():
    x, cand, conn, raw, _ = _problem(orc.GATE16, 6, 9, 8, 3)
    x = x.to(DEV).requires_grad_()
    (g,) = torch.autograd.grad(ops.fc_layer8(x, cand.to(DEV), conn.to(DEV), raw.to(DEV), orc.GATE16).sum(), [x],
                               create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [x])


def test_sizes_past_32_bit_offsets():
    """2.2e9 values packed, and a layer over 2.2e9 inputs: the last samples as in a call of their own."""
    B, D = 270001, 8190
    x = torch.rand(B, D, device=DEV)
    codes, rows = sl.pack_rows8(x)
    part = slice(B - B % 4 - 8, B)
    c, r = sl.pack_rows8(x[part])
    assert torch.equal(codes[-c.shape[0]:], c) and torch.equal(rows[part], r)
    assert torch.equal(sl.unpack_rows8(codes, rows)[part], sl.unpack_rows8(c, r))
    _, cand, conn, raw, gy = _problem(orc.GATE16, B, D, 40, 2, x=torch.zeros(1))
    y, gx, _, _ = _grads(x, cand, conn, raw, gy, orc.GATE16, 1.0)
    ys, gs, _, _ = _grads(x[part], cand, conn, raw, gy[part], orc.GATE16, 1.0)
    assert torch.equal(y[part], ys)
    assert (gx[part] - gs).abs().max() <= 64 * orc.EPS * gs.abs().max()   # one order or another of an input's sum
