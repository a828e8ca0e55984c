"""The operators on logits against their definitions in 64 bits: largest logits, draws, the loss against a teacher."""
import math

import pytest
import torch

import logits_oracle as orc
import silogic_amd as sl

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [1, 2, 3, 7, 63, 64, 65, 100, 255, 256, 257, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 5003, 20011]


def _rows(N, V, seed=0, dtype=torch.float32, kind="logits"):
    g = torch.Generator().manual_seed(seed * 7919 + N * 31 + V)
    if kind == "equal":
        x = torch.full((N, V), 0.25)
    elif kind == "counts":
        x = torch.round(10 + 3 * torch.randn(N, V, generator=g))
    elif kind == "rising":
        x = torch.arange(V).float().expand(N, V) * (20.0 / V)
    elif kind == "falling":
        x = -torch.arange(V).float().expand(N, V) * (20.0 / V)
    elif kind == "close":   # neighbours that 32 bits just tell apart
        x = 1.0 + torch.randint(0, 200, (N, V), generator=g).float() * 2.0 ** -23
    elif kind == "wide":
        x = torch.randn(N, V, generator=g) * torch.exp(10 * torch.randn(N, V, generator=g))
        x = x.clamp(-6e4, 6e4)
    else:
        x = 2.5 * torch.randn(N, V, generator=g)
        x[:, :: max(1, V // 9)] += 5 * torch.rand(x[:, :: max(1, V // 9)].shape, generator=g)
    return x.to(dtype)


KINDS = ["logits", "equal", "counts", "rising", "falling", "close", "wide"]


# ---------------------------------------------------------------------------
# largest logits
# ---------------------------------------------------------------------------
def _check_top(x, k, on=None):
    x = x.to(DEV) if on is None else on
    values, ids = sl.top_logits(x, k)
    v, i = orc.top(x, k)
    assert values.dtype == x.dtype and ids.dtype == torch.int64
    assert torch.equal(ids.cpu(), i), (k, (ids.cpu() != i).nonzero()[:4])
    assert torch.equal(values.cpu().to(orc.F64), v)


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_top_sizes(V, dtype):
    for k in sorted({1, min(V, 2), min(V, 8), min(V, 64), min(V, 65), min(V, 257), min(V, 1024)}):
        _check_top(_rows(3, V, dtype=dtype), k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [50, 300, 3000, 30000])
def test_top_kinds(kind, V):
    for dtype in TYPES:
        for k in (1, 40, min(V, 300), min(V, 1024)):
            _check_top(_rows(3, V, 1, dtype, kind), k)


def test_top_of_rows_with_absent_tokens():
    x = _rows(6, 700)
    x[0] = -INF
    x[1] = NAN
    x[2, 5:] = -INF
    x[3, ::2] = NAN
    x[4, 3], x[4, 600] = INF, INF
    x[5] = INF
    for k in (1, 6, 600, 700):
        _check_top(x, k)
    x = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0, 1e-45, -1e-45]])
    _check_top(x, 7)
    assert sl.top_logits(x.to(DEV), 7)[1].tolist() == [[5, 0, 1, 2, 3, 6, 4]]


def test_top_of_a_long_row_of_few_values():
    x = torch.randint(0, 2, (2, 150000), generator=torch.Generator().manual_seed(3)).float()
    _check_top(x, 1000)
    x[0] = 1.0
    _check_top(x, 64)


def test_top_views_shapes_and_empty():
    x = _rows(24, 500).to(DEV)
    for v in (x[:, 1:], x[::2], x[3:4], x.t(), x[:, ::3], x[:1].expand(5, -1), x.view(2, 3, 4, 500), x.view(2, 12, 500)[:, ::2, 7:],
              x[0], x.t()[5]):
        _check_top(None, 5, on=v)
    for shape in ((0, 7), (2, 0, 7)):
        values, ids = sl.top_logits(torch.empty(shape, device=DEV), 3)
        assert values.shape == ids.shape == (*shape[:-1], 3)


# ---------------------------------------------------------------------------
# draws
# ---------------------------------------------------------------------------
LIMITS = [dict(), dict(t=0.7), dict(k=1), dict(k=3), dict(k=50), dict(k=300), dict(k=2000), dict(p=0.5), dict(p=0.9, t=1.3), dict(p=0.999),
          dict(p=0.0), dict(m=0.05), dict(m=1.0), dict(k=40, p=0.8), dict(p=0.7, m=0.1), dict(k=500, m=0.02),
          dict(k=30, p=0.95, m=0.05, t=0.8), dict(t=0.0), dict(t=1e-30), dict(t=1e30), dict(t=INF), dict(t=25.0)]


def _check_sample(x, u=None, mask=None, on=None, **limits):
    x = x if on is None else on
    if u is None:
        u = torch.rand(x.shape[:-1], generator=torch.Generator().manual_seed(11))
    names = dict(t="temperature", k="top_k", p="top_p", m="min_p")
    at = lambda v: v.to(DEV) if torch.is_tensor(v) else v  # noqa: E731
    got = sl.sample_logits(x.to(DEV), u.to(DEV), mask=at(mask), **{names[n]: at(v) for n, v in limits.items()})
    assert got.dtype == torch.int64 and got.shape == x.shape[:-1]
    flat = x.reshape(-1, x.shape[-1])
    if mask is not None:
        mask = mask.expand(x.shape).reshape(flat.shape)
    want = orc.sample(flat, u.reshape(-1), mask=mask, **{n: v.reshape(-1) if torch.is_tensor(v) else v for n, v in limits.items()})
    got = got.reshape(-1).cpu()
    assert torch.equal(got, want), (limits, [(int(n), int(got[n]), int(want[n])) for n in (got != want).nonzero()[:5]])


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_sample_sizes(V, dtype):
    for limits in LIMITS:
        _check_sample(_rows(9, V, 2, dtype), **limits)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [50, 300, 3000, 30000])
def test_sample_kinds(kind, V):
    for dtype in TYPES:
        x = _rows(5, V, 3, dtype, kind)
        for limits in LIMITS[::2] if V == 30000 else LIMITS:
            _check_sample(x, **limits)


@pytest.mark.parametrize("V", [10, 64, 300, 5000])
def test_sample_random_numbers_at_their_ends(V):
    x = _rows(8, V, 4)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, -0.5, 7.0, NAN, 2.0 ** -30, 0.5])
    for limits in LIMITS:
        _check_sample(x, u, **limits)


@pytest.mark.parametrize("V", [4, 64, 100, 1000, 4096, 8000])
def test_sample_borders_between_equal_tokens(V):
    """Equal masses: the token is floor(u n) of the n that are kept, exactly, and p n of them are kept."""
    x = torch.zeros(V + 1, V)
    u = torch.arange(V + 1).float() / V
    n = torch.arange(V + 1).clamp(max=V - 1)
    for dtype in TYPES:
        y = x.to(dtype).to(DEV)
        # u V is rounded to u's 24 bits: just under a whole number it is the token before
        want = (u.double() * V).floor().long().clamp(max=V - 1)
        assert torch.equal(sl.sample_logits(y, u.to(DEV)).cpu(), want)
        if V & (V - 1) == 0:
            assert torch.equal(want, n)
        half = sl.sample_logits(y, torch.full((V + 1,), 1 - 2.0 ** -24, device=DEV), top_p=0.5)
        assert half.eq((V + 1) // 2 - 1).all()
    _check_sample(x[:8], p=0.25)
    _check_sample(x[:8], k=V // 2, p=0.5)


@pytest.mark.parametrize("V", [60, 700, 9000])
def test_sample_masks(V):
    x = _rows(12, V, 5)
    g = torch.Generator().manual_seed(V)
    mask = torch.rand(12, V, generator=g) < 0.3
    mask[0] = False
    mask[1] = False
    mask[1, V - 1] = True
    mask[2] = True
    x[3, ~mask[3]] = NAN
    x[4, ~mask[4]] = INF
    for limits in LIMITS:
        _check_sample(x, mask=mask, **limits)
    _check_sample(x, mask=mask[5])
    _check_sample(x, mask=torch.zeros(V, dtype=torch.bool))
    wide = torch.rand(12, 2 * V, generator=g) < 0.5
    _check_sample(x, mask=wide[:, ::2])
    _check_sample(x, mask=wide[:, 3:V + 3])
    _check_sample(x.view(3, 4, V), mask=mask[:4])
    _check_sample(x.view(3, 4, V), mask=mask.view(3, 4, V)[:, :1])


@pytest.mark.parametrize("V", [40, 700, 6000])
def test_sample_rows_that_are_not_finite(V):
    x = _rows(8, V, 6)
    x[0] = -INF
    x[1] = NAN
    x[2, V // 2:] = -INF
    x[3, ::3] = NAN
    x[4, [2, V - 1]] = INF
    x[5] = INF
    x[6, :] = -INF
    x[6, 7] = -3e38
    x[7, 0], x[7, 1] = 3e38, -3e38
    for limits in LIMITS:
        _check_sample(x, **limits)


@pytest.mark.parametrize("V", [30, 257, 2000, 30000])
def test_sample_limits_of_each_row(V):
    N = 40
    g = torch.Generator().manual_seed(V)
    r = torch.rand(4, N, generator=g)
    t = torch.where(r[0] < 0.2, 0.0, 2 * r[0])
    k = torch.where(r[1] < 0.5, 0, (r[1] * 1.5 * V).long())
    p = torch.where(r[2] < 0.4, 1.0, r[2])
    m = torch.where(r[3] < 0.6, 0.0, r[3] * 0.3)
    t[1], t[2], k[3], k[4], p[5], p[6], m[7], m[8] = -1.0, NAN, -5, 1 << 40, -0.5, 3.0, -1.0, 2.0
    x = _rows(N, V, 7)
    _check_sample(x, t=t, k=k, p=p, m=m)
    _check_sample(x, t=t, k=5)
    _check_sample(x, p=p)
    _check_sample(x, k=k.int(), m=m.double())
    _check_sample(x.view(5, 8, V), t=t.view(5, 8), p=p.view(5, 8))


def test_sample_views_shapes_and_empty():
    x = _rows(24, 500, 8).to(DEV)
    for v in (x[:, 1:], x[::2], x[3:4], x.t(), x[:, ::3], x[:1].expand(5, -1), x.view(2, 3, 4, 500), x.view(2, 12, 500)[:, ::2, 7:],
              x[0], x.t()[5]):
        _check_sample(None, on=v, p=0.8)
    u = torch.rand(24, 2, generator=torch.Generator().manual_seed(1))
    _check_sample(x.cpu(), u[:, 0])
    _check_sample(x.cpu(), u[:, 1].double())
    assert sl.sample_logits(torch.empty(0, 5, device=DEV), torch.empty(0, device=DEV)).shape == (0,)
    assert sl.sample_logits(torch.empty(3, 0, 5, device=DEV), torch.empty(3, 0, device=DEV)).shape == (3, 0)


def test_sample_draws_by_the_masses():
    """Shares of a fine grid of random numbers: each token as often as its probability, to one of the grid."""
    x = _rows(1, 12, 9)
    u = torch.arange(4096).float() / 4096
    got = sl.sample_logits(x.to(DEV).expand(4096, -1), u.to(DEV), temperature=0.9).cpu()
    share = torch.bincount(got, minlength=12).double() / 4096
    assert (share - torch.softmax(x[0].double() / 0.9, 0)).abs().max() <= 1 / 4096 + 1e-6


def test_sample_the_same_on_every_call():
    x, u = _rows(64, 30000, 10).to(DEV), torch.rand(64, device=DEV)
    for limits in (dict(), dict(top_p=0.95), dict(top_k=700), dict(top_p=0.9, min_p=0.01)):
        first = sl.sample_logits(x, u, **limits)
        for _ in range(4):
            assert torch.equal(sl.sample_logits(x, u, **limits), first)


# ---------------------------------------------------------------------------
# the loss against a teacher
# ---------------------------------------------------------------------------
def _teacher(x, K, seed, dtype, absent=True):
    g = torch.Generator().manual_seed(seed)
    N, V = x.shape
    t = x.float() + 2 * torch.randn(N, V, generator=g)
    values, ids = torch.topk(torch.where(t.isfinite(), t, torch.full_like(t, -50.0)), K, dim=1)
    if absent:
        drop = torch.rand(N, K, generator=g) < 0.15
        ids = torch.where(drop, torch.randint(0, 3, (N, K), generator=g) * (V + 5) - 1, ids)
        ids = torch.where((ids >= 0) & (ids < V) & drop, torch.full_like(ids, -1), ids)
        ids[N // 2] = -1
    labels = torch.where(torch.rand(N, generator=g) < 0.8, ids[:, 0], torch.randint(0, V, (N,), generator=g))
    if absent:
        labels[N // 2] = -100
        labels[0] = V
    return values.to(dtype), ids, labels


def _check_distill(x, values, ids, labels, T=1.0, alpha=0.3, reduction="mean", upstream=None, what=""):
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    lead = x.shape[:-1]
    flat = lambda t: None if t is None else t.reshape(-1, *t.shape[len(lead):])  # noqa: E731
    args = (d(values), d(ids), d(labels), T, alpha, reduction)
    s = d(x).detach().requires_grad_()
    loss = sl.distill_loss(s, *args)
    assert loss.dtype == torch.float32
    (g,) = torch.autograd.grad(loss, [s], None if upstream is None else d(upstream)) if reduction != "none" or upstream is not None \
        else torch.autograd.grad(loss.sum(), [s])
    assert g.dtype == x.dtype and g.shape == x.shape
    up = upstream if upstream is None or upstream.dim() == 0 else flat(upstream)
    want = orc.distill(flat(x), flat(values), flat(ids), flat(labels), T, alpha, reduction, up)
    what = f"{what} V={x.shape[-1]} K={values.shape[-1]} {x.dtype} T={T} {reduction}"
    orc.check_distill(loss.reshape(-1) if reduction == "none" else loss, g.reshape(-1, x.shape[-1]), want, what)
    with torch.no_grad():
        assert torch.equal(sl.distill_loss(s, *args), loss.detach())
    both = sl.distill_loss_and_grad(s, *args, scale=0.5)
    want = orc.distill(flat(x), flat(values), flat(ids), flat(labels), T, alpha, reduction, torch.tensor(0.5))
    orc.check_distill(both[0].reshape(-1) if reduction == "none" else both[0], both[1].reshape(-1, x.shape[-1]), want, what + " both")
    return loss.detach(), g


@pytest.mark.parametrize("V", SIZES + [70001])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_sizes(V, dtype):
    N = 7
    x = _rows(N, V, 12, dtype)
    for K in sorted({1, min(V, 5), min(V, 64), min(V, 300)}):
        values, ids, labels = _teacher(x, K, V + K, dtype)
        for T, with_labels, reduction in ((1.0, False, "mean"), (2.0, True, "mean"), (1.0, True, "sum"), (0.5, False, "none"),
                                          (4.0, True, "none")):
            up = torch.rand(N, generator=torch.Generator().manual_seed(K)) if reduction == "none" else None
            _check_distill(x, values, ids, labels if with_labels else None, T, 0.3, reduction, up)


@pytest.mark.parametrize("kind", ["equal", "counts", "rising", "falling", "close", "wide"])
def test_distill_kinds(kind):
    for V in (100, 9001):
        x = _rows(4, V, 13, torch.float32, kind)
        values, ids, labels = _teacher(x, 30, 5, torch.float32)
        for T in (1.0, 3.0):
            _check_distill(x, values, ids, labels, T, what=kind)


def test_distill_most_rows_and_entries():
    x = _rows(2500, 40, 14)
    values, ids, labels = _teacher(x, 8, 6, torch.float32)
    _check_distill(x, values, ids, labels, 2.0)
    _check_distill(x, values, ids, None, 2.0, reduction="none", upstream=torch.randn(2500))
    x = _rows(3, 3000, 15)
    values, ids, labels = _teacher(x, 1024, 7, torch.float32)
    _check_distill(x, values, ids, labels, 2.0)


@pytest.mark.parametrize("V", [20, 300, 20000])
def test_distill_tokens_named_twice(V):
    x = _rows(5, V, 16)
    ids = torch.randint(0, min(V, 6), (5, 40), generator=torch.Generator().manual_seed(1))
    ids[1] = V - 1
    values = torch.randn(5, 40, generator=torch.Generator().manual_seed(2))
    labels = ids[:, 3].clone()
    for labels_ in (labels, None):
        for reduction in ("sum", "none"):
            _check_distill(x, values, ids, labels_, 1.5, reduction=reduction)


@pytest.mark.parametrize("V", [20, 300, 20000])
def test_distill_masked_students_and_absent_teachers(V):
    x = _rows(8, V, 17)
    values, ids, labels = _teacher(x, 10, 3, torch.float32, absent=False)
    x[0] = -INF                          # nothing
    x[1, V // 2:] = -INF                 # masked logits, some named by the teacher
    ids[1] = torch.arange(10) % (V // 2)
    labels[1] = 0
    ids[2] = -1                          # label alone
    labels[3] = -100                     # teacher alone
    ids[4], labels[4] = V, -100          # nothing; whatever is there is not read into the result
    x[4] = NAN
    values[5, 3:] = -INF                 # entries without a value
    ids[6, 5:] = -7
    values[6, 5:] = NAN                  # NaN in absent places
    values[7] = -INF
    for T, reduction in ((1.0, "mean"), (2.0, "sum"), (1.0, "none")):
        for lab in (labels, None):
            _, g = _check_distill(x, values, ids, lab, T, reduction=reduction)
            assert not g[0].any() and not g[4].any()
    x[2, 0] = NAN                        # a row that learns shows its NaN
    loss = sl.distill_loss(x.to(DEV), values.to(DEV), ids.to(DEV), labels.to(DEV), reduction="none")
    assert loss.isnan().tolist() == [False, False, True, False, False, False, False, False]
    s = x.to(DEV).requires_grad_()
    weight = torch.ones(8, device=DEV)
    weight[2] = 0.0                      # unless it counts nothing
    (g,) = torch.autograd.grad(sl.distill_loss(s, values.to(DEV), ids.to(DEV), labels.to(DEV), reduction="none"), [s], weight)
    assert torch.isfinite(g).all() and not g[2].any()


def test_distill_where_the_student_rules_out_what_the_teacher_says():
    x = torch.tensor([[0.0, -INF, 1.0]])
    ids, values = torch.tensor([[1, 2]]), torch.tensor([[0.0, 1.0]])
    s = x.to(DEV).requires_grad_()
    loss = sl.distill_loss(s, values.to(DEV), ids.to(DEV))
    assert float(loss) == INF
    (g,) = torch.autograd.grad(loss, [s])
    q, p = torch.softmax(values[0].double(), 0), torch.softmax(x[0].double(), 0)
    want = p - torch.tensor([0.0, q[0], q[1]], dtype=orc.F64)
    assert (g[0].cpu().double() - want).abs().max() < 32 * orc.EPS


def test_distill_of_nothing():
    for N, V in ((0, 5), (4, 9)):
        x = torch.randn(N, V, device=DEV, requires_grad=True)
        values, ids = torch.randn(N, 3, device=DEV), torch.full((N, 3), -1, device=DEV)
        for reduction in ("mean", "sum", "none"):
            loss = sl.distill_loss(x, values, ids, reduction=reduction)
            assert loss.shape == ((N,) if reduction == "none" else ()) and not loss.any()
            (g,) = torch.autograd.grad(loss.sum(), [x])
            assert g.shape == x.shape and not g.any()
            both = sl.distill_loss_and_grad(x, values, ids, reduction=reduction)
            assert not both[0].any() and not both[1].any()


def test_distill_types_of_ids_and_values():
    x = _rows(6, 500, 18, torch.bfloat16)
    values, ids, labels = _teacher(x, 12, 3, torch.float32)
    for vt in TYPES:
        for it in (torch.int32, torch.int64):
            _check_distill(x, values.to(vt), ids.to(it), labels.to(it), 2.0)


def test_distill_views_and_shapes():
    x = _rows(24, 500, 19)
    values, ids, labels = _teacher(x, 12, 4, torch.float32)
    a = sl.distill_loss(x.to(DEV), values.to(DEV), ids.to(DEV), labels.to(DEV), reduction="none")
    b = sl.distill_loss(x.to(DEV).t().contiguous().t(), values.to(DEV).t().contiguous().t(), ids.to(DEV).t().contiguous().t(),
                        labels.to(DEV), reduction="none")
    assert torch.equal(a, b)
    pad = torch.zeros(24, 517, device=DEV)
    pad[:, 3:503] = x.to(DEV)
    s = pad.requires_grad_()
    loss = sl.distill_loss(s[:, 3:503], values.to(DEV), ids.to(DEV), labels.to(DEV), reduction="none")
    assert torch.equal(a, loss)
    (g,) = torch.autograd.grad(loss.sum(), [s])
    t = x.to(DEV).requires_grad_()
    (h,) = torch.autograd.grad(sl.distill_loss(t, values.to(DEV), ids.to(DEV), labels.to(DEV), reduction="none").sum(), [t])
    assert torch.equal(g[:, 3:503], h) and not g[:, :3].any() and not g[:, 503:].any()
    _check_distill(x.view(2, 3, 4, 500), values.view(2, 3, 4, 12), ids.view(2, 3, 4, 12), labels.view(2, 3, 4), reduction="none",
                   upstream=torch.rand(2, 3, 4))
    _check_distill(x[3], values[3], ids[3], labels[3], reduction="sum")
    _check_distill(x.view(4, 6, 500), values.view(4, 6, 12), ids.view(4, 6, 12), None, upstream=torch.tensor(3.0))


def test_distill_gradient_against_differences():
    x, T, alpha = _rows(3, 9, 20).double(), 1.7, 0.4
    values, ids, labels = _teacher(x.float(), 4, 8, torch.float32, absent=False)
    ids[1, 2] = ids[1, 0]
    s = x.float().to(DEV).requires_grad_()
    (g,) = torch.autograd.grad(sl.distill_loss(s, values.to(DEV), ids.to(DEV), labels.to(DEV), T, alpha), [s])
    h = 1e-5
    for n in range(3):
        for i in range(9):
            hi, lo = x.clone(), x.clone()
            hi[n, i] += h
            lo[n, i] -= h
            a, b = (float(orc.distill(v, values, ids, labels, T, alpha, "mean")["loss"]) for v in (hi, lo))
            # the difference's own error: a third derivative of size about 1 times h^2, and 2^-52 / h of rounding
            assert abs(float(g[n, i]) - (a - b) / (2 * h)) < 1e-9 + 64 * orc.EPS


def test_distill_the_same_bits_on_every_call():
    x = _rows(200, 9000, 21, torch.bfloat16).to(DEV)
    values, ids, labels = (t.to(DEV) for t in _teacher(x.cpu(), 64, 9, torch.bfloat16))
    first = sl.distill_loss_and_grad(x, values, ids, labels, 2.0)
    for _ in range(3):
        again = sl.distill_loss_and_grad(x, values, ids, labels, 2.0)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_distill_backward_twice_and_through_a_network():
    x = _rows(16, 300, 22).to(DEV).requires_grad_()
    values, ids, labels = (t.to(DEV) for t in _teacher(x.detach().cpu(), 9, 9, torch.float32))
    loss = sl.distill_loss(x, values, ids, labels, 2.0)
    (a,) = torch.autograd.grad(loss, [x], retain_graph=True)
    (b,) = torch.autograd.grad(2 * loss, [x])
    assert torch.equal(2 * a, b)   # a factor of two rounds nothing
    with pytest.raises(RuntimeError):
        (c,) = torch.autograd.grad(sl.distill_loss(x, values, ids), [x], create_graph=True)
        c.sum().backward()
