"""The token encoder's hard bits follow its weight: replaced by a view or by another width, updated by a graph."""
import pytest
import torch

import silogic_amd as sl
from silogic_amd import derived

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _packed(bits):
    """uint8 [B, F] -> words [F, ceil(B/64)]."""
    B, F = bits.shape
    rows = torch.zeros((-(-B // 64) * 64, F), device=bits.device, dtype=torch.int64)
    rows[:B] = bits
    return (rows.view(-1, 64, F) << torch.arange(64, device=bits.device).view(1, 64, 1)).sum(1).t()


def _check(enc):
    """Ids of the first table of ten rows, some of them without a row now."""
    ids = torch.arange(10, device=DEV)
    want = torch.zeros((10, enc.bits), device=DEV, dtype=torch.uint8)
    want[:enc.num_tokens] = (enc.weight > 0)
    assert torch.equal(enc.forward_hard(ids), want)
    assert torch.equal(enc.forward_packed(ids), _packed(want))
    assert torch.equal(enc.forward_packed(ids, word_major=True), _packed(want).t())


@pytest.mark.parametrize("how", ["prefix", "columns", "transposed", "type", "counter of its own"])
def test_a_weight_replaced_by_a_view_of_it(how):
    enc = sl.TokenEncoder(10, 10).to(DEV)
    _check(enc)
    w = enc.weight
    enc.weight = torch.nn.Parameter({"prefix": lambda: w.detach()[:2], "columns": lambda: w.detach()[:, :2],
                                     "transposed": lambda: w.detach().t(),
                                     "type": lambda: w.detach().view(torch.float16)[:, 1::2],
                                     "counter of its own": lambda: w.data}[how]())
    _check(enc)


@pytest.mark.parametrize("before,after", [(128, 64), (64, 65), (200, 3), (3, 200)])
def test_a_weight_of_another_width(before, after):
    enc = sl.TokenEncoder(10, before).to(DEV)
    _check(enc)
    enc.weight = torch.nn.Parameter(torch.randn(10, after, device=DEV))
    _check(enc)
    enc.ste = True
    assert torch.equal(enc(torch.arange(10, device=DEV)), (enc.weight > 0).float())


def test_a_graph_that_updates_the_weight():
    """Its replays count no version: derived.clear drops the words of the weight as it was."""
    enc = sl.TokenEncoder(10, 70).to(DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, stream=side):
        enc.weight.neg_()
    for _ in range(3):
        _check(enc)
        graph.replay()
        derived.clear(enc)
        _check(enc)
        torch.cuda.synchronize()


def test_operators_want_their_tensors_on_the_gpu():
    op = torch.ops.silogic_hip
    ids, table, gy = torch.zeros((2, 3), dtype=torch.int64), torch.rand(4, 5), torch.rand(2, 15)
    on = [t.to(DEV) for t in (ids, table, gy)]
    assert op.token_encode_bwd(on[0], on[1], 1.0, -1, on[2]).shape == (4, 5)
    for i, t in enumerate((ids, table, gy)):
        args = on[:i] + [t] + on[i + 1:]
        with pytest.raises(RuntimeError, match="GPU"):
            op.token_encode_bwd(args[0], args[1], 1.0, -1, args[2])


def test_a_stream_waits_for_the_words_of_another():
    """The words are made on the main stream behind work of some milliseconds; the side stream is idle and has
    waited for nothing since."""
    enc = sl.TokenEncoder(3000, 200).to(DEV)
    ids = torch.randint(0, 3000, (500, 4), device=DEV)
    a, b = torch.rand(2, 1 << 28, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        enc.forward_packed(ids)   # memory of the side stream's own
    for k in range(3):
        torch.cuda.synchronize()
        for _ in range(20):
            b.copy_(a)
        with torch.no_grad():
            enc.weight.neg_()
        mine = enc.forward_packed(ids)
        with torch.cuda.stream(side):
            other = enc.forward_packed(ids)
        torch.cuda.synchronize()
        want = _packed((enc.weight > 0)[ids].reshape(500, -1))
        assert torch.equal(mine, want) and torch.equal(other, want), f"call {k}"
