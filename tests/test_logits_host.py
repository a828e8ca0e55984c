"""Refusals of the operators on logits: none of these calls reaches a GPU."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import silogic_amd as sl
from silogic_amd import _lib, ops

P = C.c_void_p(16)   # an address that is only looked at
ARG, SHAPE = -1, -2
NAN = math.nan


def _entry(name, **defaults):
    return lambda **k: getattr(_lib.lib(), name)(*{**defaults, **k}.values())


def test_top_logits_entry_point():
    top = _entry("slg_top_logits", x=P, dtype=0, N=4, V=50, ld=50, K=5, values=P, ids=P, stream=None)
    for kw in (dict(x=None), dict(values=None), dict(ids=None), dict(dtype=3), dict(dtype=-1)):
        assert top(**kw) == ARG, kw
    for kw in (dict(N=-1), dict(N=1 << 31), dict(V=0), dict(V=(1 << 24) + 1), dict(K=0), dict(K=51), dict(K=1025, V=5000), dict(ld=-1)):
        assert top(**kw) == SHAPE, kw
    assert top(N=0, x=None, values=None, ids=None) == 0


def test_sample_logits_entry_point():
    draw = _entry("slg_sample_logits", x=P, dtype=0, N=4, V=50, ld=50, allowed=None, allowed_ld=0, u=P, t=1.0, k=0, p=1.0, m=0.0, ts=None,
                  ks=None, ps=None, ms=None, ids=P, stream=None)
    for kw in (dict(x=None), dict(u=None), dict(ids=None), dict(dtype=3), dict(t=-1.0), dict(t=NAN), dict(k=-1), dict(p=1.1), dict(p=NAN),
               dict(m=-0.1), dict(m=NAN)):
        assert draw(**kw) == ARG, kw
    for kw in (dict(N=-1), dict(N=1 << 31), dict(V=0), dict(V=(1 << 24) + 1), dict(ld=-1), dict(allowed_ld=-1)):
        assert draw(**kw) == SHAPE, kw
    assert draw(N=0, x=None, u=None, ids=None) == 0


def test_distill_entry_points():
    given = dict(x=P, dtype=0, N=4, V=50, ld=50, values=P, vtype=0, ids=P, id_bytes=8, K=5, labels=P, label_bytes=8, T=1.0, alpha=0.5,
                 reduction=2)
    fwd = _entry("slg_distill_fwd", **given, loss=P, kept=P, stream=None)
    bwd = _entry("slg_distill_bwd", **given, kept=P, up=P, scale=1.0, grad=P, stream=None)
    both = _entry("slg_distill_loss_grad", **given, scale=1.0, loss=P, grad=P, kept=P, stream=None)
    for call in (fwd, bwd, both):
        for kw in (dict(x=None), dict(values=None), dict(ids=None), dict(kept=None), dict(dtype=3), dict(vtype=-1), dict(id_bytes=2),
                   dict(label_bytes=1), dict(T=0.0), dict(T=NAN), dict(T=1e5), dict(alpha=-0.1), dict(alpha=NAN), dict(reduction=3)):
            assert call(**kw) == ARG, kw
        for kw in (dict(N=-1), dict(N=1 << 31), dict(V=0), dict(V=1 << 31), dict(K=0), dict(K=1025), dict(ld=-1)):
            assert call(**kw) == SHAPE, kw
    assert fwd(kept=C.c_void_p(20)) == ARG and bwd(kept=C.c_void_p(20)) == ARG and both(kept=C.c_void_p(20)) == ARG
    assert fwd(loss=None) == ARG and bwd(grad=None) == ARG and both(loss=None) == ARG
    assert both(grad=None) == ARG and both(scale=math.inf) == ARG
    assert bwd(N=0, x=None, values=None, ids=None, kept=None, grad=None) == 0
    assert fwd(N=0, reduction=0, x=None, values=None, ids=None, kept=None, loss=None) == 0
    assert [_lib.lib().slg_distill_kept(n) for n in (-1, 1 << 31)] == [-1, -1]
    for n in (0, 1, 7, 4096, (1 << 31) - 1):
        assert _lib.lib().slg_distill_kept(n) == ops.distill_kept(n)


def test_top_logits_refuses():
    x = torch.randn(3, 20)
    for k in (0, 21, -1):
        with pytest.raises(ValueError):
            sl.top_logits(x, k)
    with pytest.raises(ValueError):
        sl.top_logits(torch.randn(1, 3000), 1025)
    with pytest.raises(TypeError):
        sl.top_logits(x.double(), 2)
    with pytest.raises(ValueError):
        sl.top_logits(torch.randn(3, 0), 1)
    with pytest.raises(ValueError):
        sl.top_logits(torch.tensor(1.0), 1)
    with pytest.raises(RuntimeError, match="GPU"):
        sl.top_logits(x, 2)


def test_sample_logits_refuses():
    x, u = torch.randn(3, 20), torch.rand(3)
    for kw in (dict(temperature=-1.0), dict(temperature=NAN), dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(top_p=NAN),
               dict(min_p=2.0), dict(min_p=NAN), dict(temperature=torch.ones(4)), dict(top_k=torch.ones(3, 1, dtype=torch.int64)),
               dict(mask=torch.ones(4, 20, dtype=torch.bool)), dict(mask=torch.ones(3, 1, 20, dtype=torch.bool))):
        with pytest.raises(ValueError):
            sl.sample_logits(x, u, **kw)
    for kw in (dict(temperature=torch.ones(3, dtype=torch.int64)), dict(top_k=torch.ones(3)), dict(top_k=torch.ones(3, dtype=torch.bool)),
               dict(mask=torch.ones(3, 20))):
        with pytest.raises(TypeError):
            sl.sample_logits(x, u, **kw)
    for bad in (torch.rand(4), torch.rand(3, 1), torch.rand(())):
        with pytest.raises(ValueError):
            sl.sample_logits(x, bad)
    with pytest.raises(TypeError):
        sl.sample_logits(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        sl.sample_logits(x.long(), u)
    with pytest.raises(ValueError):
        sl.sample_logits(torch.empty(1, 1).expand(3, (1 << 24) + 1), u)
    with pytest.raises(RuntimeError, match="GPU"):
        sl.sample_logits(x, u)


@pytest.mark.parametrize("call", [sl.distill_loss, sl.distill_loss_and_grad])
def test_distill_refuses(call):
    x, v, i, y = torch.randn(3, 20), torch.randn(3, 4), torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)
    for args, kw in (((x, v[:2], i[:2]), {}), ((x, v, i[:, :2]), {}), ((x, v[0], i[0]), {}), ((x, v[:, :0], i[:, :0]), {}),
                     ((x, torch.randn(3, 1025), torch.zeros(3, 1025, dtype=torch.int64)), {}), ((x, v, i, y[:2]), {}),
                     ((x, v, i, y[:, None]), {}), ((x, v, i), dict(temperature=0.0)), ((x, v, i), dict(temperature=NAN)),
                     ((x, v, i), dict(temperature=1e6)), ((x, v, i, y), dict(alpha=1.5)), ((x, v, i, y), dict(alpha=NAN)),
                     ((x, v, i), dict(reduction="batchmean")), ((x[:, :0], v, i), {})):
        with pytest.raises(ValueError):
            call(*args, **kw)
    for args in ((x.double(), v, i), (x, v.double(), i), (x, v, i.short()), (x, v, i.float()), (x, v, i, y.float())):
        with pytest.raises(TypeError):
            call(*args)
    with pytest.raises(RuntimeError, match="GPU"):
        call(x, v, i)


def test_the_scale_is_finite():
    x, v, i = torch.randn(3, 20), torch.randn(3, 4), torch.zeros(3, 4, dtype=torch.int64)
    for scale in (NAN, math.inf):
        with pytest.raises(ValueError):
            sl.distill_loss_and_grad(x, v, i, scale=scale)


def test_limits_are_numbers_of_any_library():
    """Those of numpy are taken as Python's are; a top_k that is no whole number is refused before anything runs."""
    x, u = torch.randn(3, 20), torch.rand(3)
    for limits in (dict(top_k=np.int64(4)), dict(top_k=4.0), dict(top_p=np.float32(0.5)), dict(temperature=np.int32(1))):
        with pytest.raises(RuntimeError, match="GPU"):
            sl.sample_logits(x, u, **limits)
    with pytest.raises(TypeError, match="whole"):
        sl.sample_logits(x, u, top_k=4.5)
