"""The token encoder's hard bits after its weight was replaced, without a GPU: entry points are recorded, not
launched."""
import ctypes

import pytest
import torch

import silogic_amd as sl
from silogic_amd import _lib, ops


@pytest.fixture
def calls(monkeypatch):
    """Names and arguments of the entry points that a call would launch."""
    made = []
    monkeypatch.setattr(ops, "require_gpu", lambda *ts: None)
    monkeypatch.setattr(ops, "call_on", lambda t, name, *args: made.append((name, args)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)   # bits of every call's own
    return made


def test_words_of_another_width_are_refused(calls):
    ids = torch.zeros((2, 3), dtype=torch.int64)
    for D, words in ((65, 1), (128, 1), (64, 2), (1, 0)):
        with pytest.raises(ValueError, match="words"):
            ops.token_encode_hard(ids, torch.zeros((5, words), dtype=torch.int64), D, -1, 2)
    assert not calls
    assert ops.token_encode_hard(ids, torch.zeros((5, 2), dtype=torch.int64), 65, -1, 2).shape == (2, 195)


@pytest.mark.parametrize("before,after", [(128, 64), (64, 65), (200, 3)])
def test_a_weight_of_another_width(calls, before, after):
    """The bits' width is the present weight's in every form, not the first one's."""
    enc = sl.TokenEncoder(4, before)
    enc.weight = torch.nn.Parameter(torch.randn(7, after))
    assert (enc.num_tokens, enc.bits) == (7, after)
    ids = torch.zeros((2, 3), dtype=torch.int64)
    assert enc.forward_hard(ids).shape == (2, 3 * after)
    assert enc.forward_packed(ids).shape == (3 * after, 1)
    for name, args in calls:
        if name == "slg_token_encode_hard":
            assert args[4:6] == (7, after)   # V, D
    assert len(calls) == 4


def test_a_weight_that_is_no_table(calls):
    enc = sl.TokenEncoder(4, 5)
    for w in (torch.randn(20), torch.randn(2, 2, 5), torch.randn(0, 5), torch.randn(5, 0)):
        enc.weight = torch.nn.Parameter(w)
        for form in (enc, enc.forward_hard, enc.forward_packed):
            with pytest.raises(ValueError, match="weight"):
                form(torch.zeros(3, dtype=torch.int64))
    assert not calls


class _Stream:
    cuda_stream = 0

    def record_event(self):
        return object()


@pytest.fixture
def made(calls, monkeypatch):
    """The weights that bit tables were made of, outside a capture."""
    tables = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: _Stream())
    monkeypatch.setattr(ops, "_stream", lambda t: type("", (), {"value": 0}))
    real = ops.token_bits
    monkeypatch.setattr(ops, "token_bits", lambda t: (tables.append(t), real(t))[1])
    return tables


# replacements that start at the old weight's address
VIEWS = {
    "prefix": lambda w: torch.nn.Parameter(w.detach()[:2]),
    "columns": lambda w: torch.nn.Parameter(w.detach()[:, :2]),
    "transposed": lambda w: torch.nn.Parameter(w.detach().t()),
    "type": lambda w: torch.nn.Parameter(w.detach().view(torch.float16)[:, :4]),
    "counter of its own": lambda w: torch.nn.Parameter(w.data),
}


@pytest.mark.parametrize("how", list(VIEWS))
def test_a_weight_replaced_by_a_view_of_it(made, how):
    enc = sl.TokenEncoder(4, 4)
    ids = torch.zeros(3, dtype=torch.int64)
    enc.forward_hard(ids)
    enc.forward_packed(ids)
    assert len(made) == 1   # one table for both
    old = enc.weight
    enc.weight = VIEWS[how](old)
    assert enc.weight.data_ptr() == old.data_ptr() and enc.weight._version == old._version
    enc.forward_hard(ids)
    enc.forward_packed(ids)
    assert len(made) == 2 and torch.equal(made[1], enc.weight)


def test_a_new_weight_of_the_same_version(made):
    """Another parameter on the same memory counts its changes by itself."""
    enc = sl.TokenEncoder(4, 4)
    ids = torch.zeros(3, dtype=torch.int64)
    with torch.no_grad():
        enc.weight.neg_()
    enc.forward_hard(ids)
    old = enc.weight
    enc.weight = torch.nn.Parameter(old.data)
    with torch.no_grad():
        enc.weight.neg_()
    assert enc.weight.data_ptr() == old.data_ptr() and enc.weight._version == old._version
    enc.forward_hard(ids)
    assert len(made) == 2


@pytest.mark.parametrize("ids,table", [(torch.zeros(2, 3), torch.rand(4, 5)), (torch.zeros(2, 3, dtype=torch.int16), torch.rand(4, 5)),
                                       (torch.zeros(3, dtype=torch.int64), torch.rand(4, 5)),
                                       (torch.zeros((2, 3), dtype=torch.int64), torch.rand(4, 5).double()),
                                       (torch.zeros((2, 3), dtype=torch.int64), torch.rand(0, 5)),
                                       (torch.zeros((2, 3), dtype=torch.int64), torch.rand(4))])
def test_operators_refuse_what_the_kernels_do_not_take(ids, table):
    with pytest.raises(ValueError, match="token encoder"):
        torch.ops.silogic_hip.token_encode(ids, table, 1.0, False, -1)
    with pytest.raises(ValueError, match="token encoder"):
        torch.ops.silogic_hip.token_encode_bwd(ids, table, 1.0, -1, torch.rand(2, 15))


def test_operators_on_the_cpu():
    ids, table = torch.zeros((2, 3), dtype=torch.int64), torch.rand(4, 5)
    with pytest.raises(RuntimeError, match="GPU"):
        torch.ops.silogic_hip.token_encode(ids, table, 1.0, False, -1)
    with pytest.raises(RuntimeError, match="GPU"):
        torch.ops.silogic_hip.token_encode_bwd(ids, table, 1.0, -1, torch.rand(2, 15))


@pytest.mark.parametrize("scale", [0.0, -0.0, -1.0, float("nan"), float("inf"), -float("inf"), 3e38])
def test_scales_that_part_the_soft_form_from_the_bits(scale):
    with pytest.raises(ValueError, match="scale"):
        sl.TokenEncoder(4, 5, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        sl.TokenEncoder.from_weight(torch.randn(4, 5), scale=scale)
    at = ctypes.c_void_p(16)   # an address that is only looked at
    lib = _lib.lib()
    assert lib.slg_token_encode(at, 8, 4, 5, 6, -1, at, 0, scale, 0, at, None) == -1
    n = lib.slg_token_encode_bwd_workspace(4, 5, 6)
    assert lib.slg_token_encode_bwd(at, 8, 4, 5, 6, -1, at, 0, scale, at, at, at, n, None) == -1


def test_another_stream_waits_for_the_words(made, monkeypatch):
    """The event of the stream that made them, before their first use on another."""
    did, now = [], ["main"]

    class Stream:
        def record_event(self):
            return ("made on", now[0])

        def wait_event(self, event):
            did.append((now[0], event))

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(ops, "_stream", lambda t: type("", (), {"value": now[0]}))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: did.append((now[0], "kept")))
    enc = sl.TokenEncoder(4, 5)
    ids = torch.zeros(3, dtype=torch.int64)
    enc.forward_hard(ids)
    enc.forward_hard(ids)
    assert not did
    now[0] = "side"
    enc.forward_hard(ids)
    assert did == [("side", ("made on", "main")), ("side", "kept")] and len(made) == 1
    with torch.no_grad():
        enc.weight.neg_()
    enc.forward_hard(ids)   # made anew, here
    assert len(did) == 2 and len(made) == 2
    now[0] = "main"
    enc.forward_hard(ids)
    assert did[2:] == [("main", ("made on", "side")), ("main", "kept")]
