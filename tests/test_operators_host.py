"""Refusals of the token encoder and of the 8-bit activations: none of these calls reaches a GPU."""
import ctypes as C

import pytest
import torch

import silogic_amd as sl
from silogic_amd import _lib, ops

P = C.c_void_p(16)   # an address that is only looked at
ARG, SHAPE = -1, -2


def _rc(name, *args):
    return getattr(_lib.lib(), name)(*args)


def test_rows8_entry_points():
    assert _rc("slg_rows8_pack", None, 4, 8, P, P, None) == ARG
    assert _rc("slg_rows8_pack", P, 4, 0, P, P, None) == SHAPE
    assert _rc("slg_rows8_pack", P, -1, 8, P, P, None) == SHAPE
    assert _rc("slg_rows8_pack", P, 1 << 31, 8, P, P, None) == SHAPE
    assert _rc("slg_rows8_pack", P, 1 << 20, 1 << 27, P, P, None) == SHAPE
    assert _rc("slg_rows8_pack", P, 4, 8, C.c_void_p(20), P, None) == ARG
    assert _rc("slg_rows8_pack", None, 0, 8, None, None, None) == 0
    assert _rc("slg_rows8_unpack", P, None, 4, 8, P, None) == ARG
    assert _rc("slg_rows8_unpack", P, P, 4, 1 << 28, P, None) == SHAPE
    assert _rc("slg_rows8_unpack", C.c_void_p(8), P, 4, 8, P, None) == ARG
    assert _rc("slg_rows8_unpack", None, None, 0, 8, None, None) == 0
    assert [_rc("slg_rows8_ld", d) for d in (1, 4, 5, 8)] == [4, 4, 8, 8]


def test_bwd8_entry_points():
    ws = _rc("slg_fc_soft_bwd8_workspace", 16, 100, 50, 4)
    assert ws > 0
    for bad in ((-1, 100, 50, 4), (16, 0, 50, 4), (16, 100, 0, 4), (16, 100, 50, 0), (16, 100, 50, 17),
                (16, 41000, 50, 4), (16, 100, 1 << 28, 4), (1 << 31, 100, 50, 4)):
        assert _rc("slg_fc_soft_bwd8_workspace", *bad) == -1, bad

    def call(codes=P, rows=P, B=16, IN=100, OUT=50, K=4, cand=P, w=P, kind=0, npar=P, gy=P, work=P, n=ws):
        return _rc("slg_fc_soft_bwd8", codes, rows, B, IN, OUT, K, cand, w, kind, npar, 1.0, gy, P, P, P, work,
                   n, None)

    for kw in (dict(codes=None), dict(rows=None), dict(cand=None), dict(w=None), dict(npar=None), dict(gy=None),
               dict(work=None), dict(kind=3), dict(kind=-1), dict(n=ws - 1), dict(codes=C.c_void_p(4)),
               dict(work=C.c_void_p(8))):
        assert call(**kw) == ARG, kw
    for kw in (dict(K=17), dict(K=0), dict(OUT=0), dict(IN=0), dict(IN=41000), dict(B=-1)):
        assert call(**kw) == SHAPE, kw


def test_token_entry_points():
    enc = lambda **k: _rc("slg_token_encode", *{**dict(ids=P, size=8, N=4, V=5, D=6, pad=-1, table=P,  # noqa: E731
                                                       dtype=0, scale=1.0, ste=0, y=P, stream=None), **k}.values())
    for kw in (dict(ids=None), dict(table=None), dict(y=None), dict(size=2), dict(dtype=3), dict(dtype=-1)):
        assert enc(**kw) == ARG, kw
    for kw in (dict(N=-1), dict(V=0), dict(D=0), dict(N=1 << 31), dict(V=1 << 30), dict(D=1 << 24),
               dict(N=1 << 30, D=1 << 20)):
        assert enc(**kw) == SHAPE, kw
    assert enc(N=0, ids=None, y=None) == 0
    ws = _rc("slg_token_encode_bwd_workspace", 1000, 50, 16)
    assert ws > 0 and _rc("slg_token_encode_bwd_workspace", 1000, 0, 16) == -1
    bwd = lambda **k: _rc("slg_token_encode_bwd", *{**dict(ids=P, size=8, N=1000, V=50, D=16, pad=-1, table=P,  # noqa: E731
                                                           dtype=0, scale=1.0, gy=P, g=P, work=P, n=ws,
                                                           stream=None), **k}.values())
    for kw in (dict(ids=None), dict(table=None), dict(gy=None), dict(g=None), dict(work=None), dict(size=1),
               dict(dtype=7), dict(n=ws - 1), dict(work=C.c_void_p(8))):
        assert bwd(**kw) == ARG, kw
    assert bwd(D=0) == SHAPE
    assert _rc("slg_token_bits", None, 0, 5, 6, P, None) == ARG
    assert _rc("slg_token_bits", P, 5, 5, 6, P, None) == ARG
    assert _rc("slg_token_bits", P, 0, 0, 6, P, None) == SHAPE
    hard = lambda **k: _rc("slg_token_encode_hard", *{**dict(ids=P, size=8, B=4, L=3, V=5, D=6, pad=-1, bits=P,  # noqa: E731
                                                             layout=0, out=P, stream=None), **k}.values())
    for kw in (dict(ids=None), dict(bits=None), dict(out=None), dict(layout=3), dict(layout=-1), dict(size=3)):
        assert hard(**kw) == ARG, kw
    for kw in (dict(B=-1), dict(L=1 << 31), dict(B=1 << 30, L=1 << 30), dict(V=0)):
        assert hard(**kw) == SHAPE, kw
    assert hard(B=0, ids=None, out=None) == 0


def test_encoder_refuses():
    with pytest.raises(ValueError):
        sl.TokenEncoder.from_weight(torch.randn(5))
    with pytest.raises(ValueError):
        sl.TokenEncoder.from_weight(torch.randn(0, 5))
    with pytest.raises(TypeError):
        sl.TokenEncoder.from_weight(torch.randn(4, 5).double())
    with pytest.raises(ValueError):
        sl.TokenEncoder(4, 5, padding_idx=4)
    enc = sl.TokenEncoder(4, 5, padding_idx=-1)
    assert enc.padding_idx == 3 and list(enc.state_dict()) == ["weight"]
    with pytest.raises(TypeError):
        enc(torch.zeros(3))
    with pytest.raises(TypeError):
        enc(torch.zeros(3, dtype=torch.int16))
    with pytest.raises(ValueError):
        enc(torch.zeros(2, 3, 4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        enc(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        sl.TokenEncoder(4, 5).double()(torch.zeros(3, dtype=torch.int64))


def test_activations_refuse():
    with pytest.raises(RuntimeError, match="GPU"):
        sl.pack_rows8(torch.rand(3, 4))
    net = sl.LogicNet(16, 20, 2, num_classes=10, k=4)
    with pytest.raises(ValueError):
        sl.save_activations(net, 4)
    assert sl.save_activations(net) == 2 and all(m.saved_bits == 8 for m in net.layers)
    assert sl.save_activations(net, 32) == 2 and all(m.saved_bits == 32 for m in net.layers)
    for model in (torch.nn.Linear(3, 4), sl.LUTkLayer(16, 20, k=4), sl.LogicLayer(40, 20, k=17)):
        with pytest.raises(ValueError):
            sl.save_activations(model)
    with pytest.raises(NotImplementedError):
        ops.check_layer8(torch.rand(2, 40), torch.zeros(5, 2, 17))
    with pytest.raises(NotImplementedError):
        ops.check_layer8(torch.rand(2, 40), torch.zeros(5, 4, 3))
    with pytest.raises(ValueError):
        ops.check_layer8(torch.rand(2), torch.zeros(5, 2, 3))
    with pytest.raises(ValueError):
        ops.check_layer8(torch.rand(2, 4), torch.zeros(5, 2, 3), w=(torch.zeros(5, 2, 2), (5, 2, 3)))
