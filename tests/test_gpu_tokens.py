"""The token encoder against 64-bit oracles: values, table gradients, hard bits, and the networks it feeds."""
import pytest
import torch

import silogic_amd as sl
import rows8_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64
# unit rounding of the gradient's type: half a step relative to the value
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _oracle(ids, table, scale, ste, pad, gy=None):
    """Values [B, L*D], bits, the table's gradient and the sums of the terms' absolute values."""
    ids = ids.long().cpu() if ids.dim() == 2 else ids.long().cpu().unsqueeze(1)
    e = table.detach().cpu().to(F64)
    V, D = e.shape
    there = (ids >= 0) & (ids < V) & (ids != (-1 if pad is None else pad))
    row = torch.where(there, ids, torch.zeros_like(ids))
    bits = (e > 0)[row] & there.unsqueeze(-1)
    y = bits.to(F64) if ste else torch.sigmoid(scale * e)[row] * there.unsqueeze(-1)
    out = [y.reshape(len(ids), -1), bits.reshape(len(ids), -1)]
    if gy is not None:
        g = gy.cpu().to(F64).reshape(*ids.shape, D) * there.unsqueeze(-1)
        slope = (scale * torch.sigmoid(scale * e) * torch.sigmoid(-scale * e))
        flat = row.reshape(-1)
        total = torch.zeros(V, D, dtype=F64).index_add_(0, flat, g.reshape(-1, D))
        size = torch.zeros(V, D, dtype=F64).index_add_(0, flat, g.abs().reshape(-1, D))
        count = torch.bincount(flat, minlength=V).to(F64)[:, None]
        out += [total * slope, (size * count) * slope.abs(), size * slope.abs()]
    return out


def _ids(B, L, V, how, g):
    if how == "uniform":
        return torch.randint(0, V, (B, L), generator=g)
    if how == "one":
        return torch.full((B, L), V // 2)
    if how == "absent":
        return torch.full((B, L), -3)
    if how == "wild":   # padding, negative ids and ids past the table among the rest
        return torch.randint(-V - 2, 3 * V + 2, (B, L), generator=g)
    u = torch.rand(B, L, generator=g)   # frequencies one over the rank
    return (torch.exp(u * torch.log(torch.tensor(float(V)))).long() - 1).clamp(0, V - 1)


def _check(B, L, V, D, how="zipf", dtype=torch.float32, ste=False, pad=None, scale=1.25, int32=False):
    g = torch.Generator().manual_seed(B * 7 + L * 5 + V * 3 + D)
    ids = _ids(B, L, V, how, g)
    table = torch.randn(V, D, generator=g).to(dtype)
    gy = torch.randn(B, L * D, generator=g)
    enc = sl.TokenEncoder.from_weight(table.to(DEV), scale=scale, ste=ste, padding_idx=pad)
    dids = ids.to(DEV).to(torch.int32 if int32 else torch.int64)
    y = enc(dids)
    (gt,) = torch.autograd.grad(y, [enc.weight], gy.to(DEV))
    yw, bits, gw, spread, size = _oracle(ids, table, scale, ste, enc.padding_idx, gy)
    z = (scale * table.to(F64).abs()).max()
    # 1 / (1 + 2^t), t = e * (scale log2 e): the factor and the product each rounded once shift t ln 2 = z by
    # at most 2 z 2^-24, which y follows by no more than that relative to it; the exponential and the
    # reciprocal are off by an ulp (2 units) each, the sum by one
    orc.close(y, yw, (2 * z + 8) * orc.EPS * yw.abs(), "values")
    assert gt.dtype == dtype and gt.shape == table.shape
    # n - 1 sums of n terms: off by at most n 2^-24 of the terms' sizes; the slope as above; the type's rounding
    # (with fp16, values under its normal range go by its smallest step, 2^-25 at most)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -149
    orc.close(gt, gw, orc.EPS * spread + (2 * z + 16) * orc.EPS * size + 1.001 * U[dtype] * gw.abs() + tiny, "gradient")
    hard = enc.forward_hard(dids)
    assert hard.dtype == torch.uint8 and torch.equal(hard.cpu().bool(), bits)
    for wm in (False, True):
        words = enc.forward_packed(dids, word_major=wm)
        want = sl.ops.pack_bits(bits.to(torch.uint8).to(DEV), wm) if B else words
        assert words.dtype == torch.int64 and torch.equal(words, want), "packed"


@pytest.mark.parametrize("B,L,V,D", [(1, 1, 1, 1), (1, 1, 2, 16), (1, 3, 5, 7), (2, 1, 300, 64), (63, 2, 17, 3),
                                     (64, 5, 100, 65), (65, 4, 1000, 32), (130, 33, 70, 10), (257, 16, 511, 24),
                                     (100, 50, 512, 4), (33, 200, 513, 130), (7, 1, 70000, 8), (5, 3, 9, 600),
                                     (300, 40, 3, 12), (513, 64, 4001, 5), (41, 7, 60, 27), (3, 3, 40, 301), (70, 3, 90, 8),
                                     (66, 9, 30, 9)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_sizes(B, L, V, D, dtype):
    _check(B, L, V, D, dtype=dtype, pad=0 if V > 1 else None)


@pytest.mark.parametrize("how", ["uniform", "one", "absent", "wild", "zipf"])
@pytest.mark.parametrize("ste", [False, True])
@pytest.mark.parametrize("int32", [False, True])
def test_ids(how, ste, int32):
    for pad in (None, 0, -1):
        _check(90, 37, 50, 20, how=how, ste=ste, pad=pad, int32=int32)


@pytest.mark.parametrize("how", ["uniform", "one", "zipf"])
def test_sorts_of_several_workgroups(how):
    """Past one workgroup's tile of the sort, with two and three digits."""
    _check(700, 30, 40, 8, how=how)
    _check(500, 41, 30000, 8, how=how, pad=5)
    _check(301, 30, 300000, 4, how=how)


@pytest.mark.parametrize("how", ["one", "zipf"])
def test_sorts_whose_counts_are_scanned_first(how):
    """More than 524288 tokens; runs over thousands of chunks."""
    _check(2100, 260, 1000, 1, how=how, int32=True)
    _check(1100, 500, 70000, 6, how=how)


def test_large_values_and_scales():
    """Saturated sigmoids: slopes of tiny size keep their relative exactness."""
    table = torch.tensor([[-60.0, -20.0, -1e-3, 0.0], [20.0, 60.0, 3e38, -3e38]])
    ids = torch.tensor([[0, 1], [1, 1], [0, 0]])
    gy = torch.randn(3, 8)
    enc = sl.TokenEncoder.from_weight(table.to(DEV))
    y = enc(ids.to(DEV))
    (gt,) = torch.autograd.grad(y, [enc.weight], gy.to(DEV))
    yw, _, gw, spread, size = _oracle(ids, table, 1.0, False, None, gy)
    z = table.to(F64).abs().clamp_max(104)   # past it exp is 0 in fp32
    zy = z[ids].reshape(3, 8)
    orc.close(y, yw, (2 * zy + 8) * orc.EPS * yw + 2.0 ** -126, "values")
    orc.close(gt, gw, orc.EPS * spread + (2 * z + 16) * orc.EPS * size + 2.0 ** -126, "gradient")


def test_entries_that_are_not_finite():
    nan, inf = float("nan"), float("inf")
    enc = sl.TokenEncoder.from_weight(torch.tensor([[nan, inf, -inf], [1.0, -1.0, 0.5]], device=DEV))
    ids = torch.tensor([0, 1], device=DEV)
    y = enc(ids)
    assert torch.isnan(y[0, 0]) and y[0, 1:].tolist() == [1.0, 0.0]
    assert enc.forward_hard(ids).tolist() == [[0, 1, 0], [1, 0, 1]]
    (g,) = torch.autograd.grad(y[1:].sum(), [enc.weight])   # the first row's upstream gradient is 0
    assert torch.isfinite(g[1]).all()


def test_padding_rows_are_never_read():
    """Absent tokens: a padding row and an upstream gradient of NaN and infinity there change nothing."""
    table = torch.randn(6, 5)
    ids = torch.tensor([[1, 0], [2, 0], [0, 0]])
    gy = torch.randn(3, 10)
    gy[2], gy[:, 5:] = float("nan"), float("inf")
    enc = sl.TokenEncoder.from_weight(table.to(DEV), padding_idx=0)
    enc.weight.data[0] = float("nan")
    y = enc(ids.to(DEV))
    assert not y[:, 5:].any() and not y[2].any()
    (g,) = torch.autograd.grad(y, [enc.weight], gy.to(DEV))
    assert not g[0].any() and not g[3:].any() and torch.isfinite(g).all()


def test_empty():
    enc = sl.TokenEncoder(7, 5).to(DEV)
    for shape in ((0,), (0, 3), (4, 0)):
        ids = torch.zeros(shape, dtype=torch.int64, device=DEV)
        y = enc(ids)
        L = shape[1] if len(shape) == 2 else 1
        assert y.shape == (shape[0], 5 * L)
        (g,) = torch.autograd.grad(y.sum(), [enc.weight])
        assert not g.any()
        assert enc.forward_hard(ids).shape == y.shape
        assert enc.forward_packed(ids).shape == (5 * L, -(-shape[0] // 64))


def test_gradient_against_differences():
    table = torch.randn(5, 3)
    ids = torch.tensor([[0, 1], [1, 1], [3, 0]])
    gy = torch.randn(3, 6)
    enc = sl.TokenEncoder.from_weight(table.to(DEV), scale=0.7)
    (g,) = torch.autograd.grad(enc(ids.to(DEV)), [enc.weight], gy.to(DEV))
    h = 1e-5
    for v in range(5):
        for d in range(3):
            hi, lo = table.to(F64), table.to(F64)
            hi[v, d] += h
            lo[v, d] -= h
            want = sum(s * float((_oracle(ids, t, 0.7, False, None)[0] * gy).sum()) for s, t in ((1, hi), (-1, lo))) / (2 * h)
            assert abs(float(g[v, d]) - want) < 1e-8 + 60 * orc.EPS


def test_views_of_ids_gradients_and_weights():
    enc = sl.TokenEncoder.from_weight(torch.randn(20, 6, device=DEV).t().contiguous().t())
    ids = torch.randint(0, 20, (8, 10), device=DEV)
    dense = sl.TokenEncoder.from_weight(enc.weight.detach().contiguous())
    for v in (ids.t(), ids[:, ::2], ids[1:, 3:], ids[:, 2]):
        a, b = enc(v), dense(v.contiguous())
        assert torch.equal(a, b)
        gy = torch.randn(a.shape[1], a.shape[0], device=DEV).t()
        assert torch.equal(torch.autograd.grad(a, [enc.weight], gy)[0],
                           torch.autograd.grad(b, [dense.weight], gy.contiguous())[0])
        assert torch.equal(enc.forward_packed(v), dense.forward_packed(v.contiguous()))


def test_the_same_bits_on_every_call():
    enc = sl.TokenEncoder(40, 33).to(DEV)
    ids = torch.randint(0, 40, (600, 20), device=DEV)
    gy = torch.randn(600, 20 * 33, device=DEV)
    first = torch.autograd.grad(enc(ids), [enc.weight], gy)[0]
    for _ in range(3):
        assert torch.equal(torch.autograd.grad(enc(ids), [enc.weight], gy)[0], first)


def test_bits_follow_the_weight():
    enc = sl.TokenEncoder(10, 70).to(DEV)
    ids = torch.arange(10, device=DEV)
    for change in (lambda: enc.weight.detach().neg_(), lambda: enc.weight.detach().mul_(-0.5),
                   lambda: setattr(enc, "weight", torch.nn.Parameter(torch.randn(10, 70, device=DEV))),
                   lambda: enc.load_state_dict({"weight": torch.randn(10, 70)})):
        assert torch.equal(enc.forward_hard(ids).bool(), enc.weight > 0)
        change()
        assert torch.equal(enc.forward_hard(ids).bool(), enc.weight > 0)
    half = enc.half()
    assert torch.equal(half.forward_hard(ids).bool(), half.weight > 0)


def test_bits_made_on_one_stream_and_read_on_another():
    enc = sl.TokenEncoder(3000, 200).to(DEV)
    ids = torch.randint(0, 3000, (500, 4), device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.no_grad():
            enc.weight.neg_()
        a = enc.forward_packed(ids)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = enc.forward_packed(ids)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, b)


def test_captured():
    """Training and packed bits in graphs, replayed between eager work; the packed call is captured before
    any eager one, and the weight changes between replays of a graph that makes its own table."""
    enc = sl.TokenEncoder(50, 20).to(DEV)
    ids = torch.randint(0, 50, (70, 6), device=DEV)
    gy = torch.randn(70, 120, device=DEV)

    def step(ids, gy):
        w = enc.weight.detach().requires_grad_()
        y = sl.encoders._TokenFn.apply(ids, w, 1.0, False, -1)
        return y, torch.autograd.grad(y, [w], gy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ids, gy)
    torch.cuda.synchronize()
    train, hard = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(train, stream=side):
        out = step(ids, gy)
    with torch.cuda.graph(hard, stream=side):
        words = enc.forward_packed(ids)
    for k in range(4):
        ids.copy_(torch.randint(0, 50, (70, 6), device=DEV))
        gy.copy_(torch.randn(70, 120, device=DEV))
        with torch.no_grad():
            enc.weight.neg_()
        train.replay()
        hard.replay()
        want = step(ids.clone(), gy.clone())
        bits = enc.forward_packed(ids.clone())
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), f"replay {k}"
        assert torch.equal(words, bits), f"replay {k}"


def test_compiled_and_checked():
    enc = sl.TokenEncoder(30, 8, padding_idx=2).to(DEV)
    ids = torch.randint(0, 30, (9, 4), device=DEV)
    y = enc(ids)
    want = torch.autograd.grad(y.sum(), [enc.weight])[0]
    c = torch.compile(enc, backend="aot_eager", fullgraph=True)(ids)
    assert torch.equal(c, y)
    assert torch.equal(torch.autograd.grad(c.sum(), [enc.weight])[0], want)
    w = torch.randn(30, 8, device=DEV, requires_grad=True)
    torch.library.opcheck(torch.ops.silogic_hip.token_encode, (ids, w, 1.5, False, 2))


def test_copies_and_pickles():
    import copy
    import io
    enc = sl.TokenEncoder(9, 70, padding_idx=1).to(DEV)
    ids = torch.arange(9, device=DEV)
    want = enc.forward_packed(ids)   # the bit table is there
    other = copy.deepcopy(enc)
    with torch.no_grad():
        other.weight.neg_()
    assert torch.equal(enc.forward_packed(ids), want)
    assert torch.equal(other.forward_hard(ids)[0].bool(), other.weight[0] > 0)
    f = io.BytesIO()
    torch.save(enc, f)
    f.seek(0)
    back = torch.load(f, weights_only=False)   # the file is this test's own
    assert torch.equal(back.forward_packed(ids), want) and back.padding_idx == 1


def test_no_second_derivative():
    enc = sl.TokenEncoder(9, 7).to(DEV)
    (g,) = torch.autograd.grad(enc(torch.arange(9, device=DEV)).sum(), [enc.weight], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [enc.weight])


def test_ids_far_outside_the_table():
    enc = sl.TokenEncoder(9, 7).to(DEV)
    ids = torch.tensor([3, 2 ** 40 + 3, -2 ** 62, 2 ** 63 - 1, -1, 9], device=DEV)
    y = enc(ids)
    assert y[0].all() and not y[1:].any() and not enc.forward_hard(ids)[1:].any()
    (g,) = torch.autograd.grad(y.sum(), [enc.weight])
    assert g[3].all() and not g[:3].any() and not g[4:].any()


def test_under_autocast():
    enc = sl.TokenEncoder(9, 7).to(DEV)
    ids = torch.arange(9, device=DEV)
    y = enc(ids)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(enc(ids), y)


def test_values_past_32_bit_offsets():
    """2.2e9 values: the last tokens' values, and counts exact in fp32 as every row's sum."""
    V, D, N = 1000, 130, 2 ** 24 + 5
    enc = sl.TokenEncoder(V, D, scale=0.5).to(DEV)
    ids = (torch.arange(N, device=DEV) * 7919) % V
    y = enc(ids)
    for part in (slice(0, 64), slice(N // 2, N // 2 + 64), slice(N - 64, N)):
        assert torch.equal(y[part], enc(ids[part]))
    (g,) = torch.autograd.grad(y, [enc.weight], torch.ones_like(y))
    count = torch.bincount(ids, minlength=V)
    (one,) = torch.autograd.grad(enc(torch.arange(V, device=DEV)).sum(), [enc.weight])
    # the sums are whole numbers below 2^24; a product's rounding each way
    orc.close(g, one.cpu().to(F64) * count.cpu().to(F64)[:, None], 2 * orc.EPS * (one.cpu().to(F64) * count.cpu()[:, None]))


def test_feeds_a_network():
    """Tokens through the encoder, gate layers that keep bytes and the head: a training step's gradients against
    the 64-bit ones at the values that each layer kept, and the circuit against the hard layers' own path."""
    torch.manual_seed(0)
    enc = sl.TokenEncoder(40, 8, padding_idx=0).to(DEV)
    net = sl.LogicNet(6 * 8, 60, 2, num_classes=10, k=4, tau=3.0, seed=0).to(DEV)
    assert sl.save_activations(net) == 2
    net.train()
    ids = torch.randint(0, 40, (100, 6), device=DEV)
    label = torch.randint(0, 10, (100,), device=DEV)
    torch.nn.functional.cross_entropy(net(enc(ids)), label).backward()
    # the same step layer by layer, for what each kept and the gradient at the head's input
    x = [enc(ids).detach()]
    for layer in net.layers:
        x.append(layer(x[-1]).detach())
    top = x[-1].clone().requires_grad_()
    (g,) = torch.autograd.grad(torch.nn.functional.cross_entropy(net.head(top), label), [top])
    g = g.cpu().to(F64)
    mag, n = g.abs(), 0
    for layer, kept in zip(reversed(list(net.layers)), (x[1], x[0])):
        cand, conn, raw = layer._conn.cand_i32, layer._conn.conn.detach().cpu(), layer.node.raw().detach().cpu()
        w = torch.softmax(conn.to(F64), -1)
        p, pmag, back, back_mag = orc.poly(orc.GATE16, raw)
        v = orc.values_of(kept)
        (_, gx, gw, gp), _ = orc.layer(v, cand, w, p, orc.GATE16, 1.0, g, pmag)
        # errors of the gradient from above go on with its mag in the place of its size
        _, (_, gxm, gwm, gpm) = orc.layer(v, cand, w, p, orc.GATE16, 1.0, mag, pmag)
        n += 4 * 4 + 80 + 100 + 2 * 4 * 60   # as in the layers' own tests, references at most all
        orc.close(layer._conn.conn.grad, orc.softmax_back(w, gw), n * orc.EPS * orc.softmax_back_mag(w, gwm), "conn")
        orc.close(layer.node.raw().grad, back(gp), n * orc.EPS * back_mag(gpm), "node")
        g, mag = gx, gxm
    _, _, want, _, _ = _oracle(ids, enc.weight, 1.0, False, 0, g)
    _, _, _, _, size = _oracle(ids, enc.weight, 1.0, False, 0, mag)
    orc.close(enc.weight.grad, want, (n + 600 + 30) * orc.EPS * size, "table")
    assert not enc.weight.grad[0].any() and enc.weight.grad[1:].any()
    net.eval()
    hard = net.forward_hard(enc.forward_hard(ids).float())
    for wm in (False, True):
        assert torch.equal(net.forward_hard_packed(enc.forward_packed(ids, word_major=wm), 100, wm), hard)


def test_a_weight_made_in_inference_mode():
    """It has no version counter: every call reads it afresh."""
    ids = torch.arange(40, device=DEV).view(8, 5) % 9
    with torch.inference_mode():
        enc = sl.TokenEncoder(9, 12).to(DEV)
        for _ in range(2):
            assert torch.equal(enc.forward_hard(ids).view(40, 12).bool(), enc.weight[ids.view(-1)] > 0)
            enc.weight.neg_()
        e = enc.weight[ids.view(-1)].double()
        want = torch.sigmoid(e)
        orc.close(enc(ids).view(40, 12), want, (2 * e.abs().max() + 8) * orc.EPS * want, "values")   # as _check
