"""The operators on logits with more rows than one dimension of a launch takes (2^32 threads), sums over many rows, and
many entries of a row that name few tokens."""
import threading

import numpy as np
import pytest
import torch

import logits_oracle as orc
import silogic_amd as sl

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS = (1 << 26) + 1000   # of workgroups of 64 threads and more


def test_rows_past_a_launch_dimension_are_listed_and_drawn():
    """The largest token, which k = 1, temperature 0 and u = 0 all give, of each of 2^26 rows and some."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(ROWS, 4, device=DEV, generator=g)
    best = x.max(1).values
    values, ids = sl.top_logits(x, 1)
    assert torch.equal(values[:, 0], best) and torch.equal(x.gather(1, ids)[:, 0], best)
    u = torch.zeros(ROWS, device=DEV)
    for t in (0.0, 1.0):
        ids = sl.sample_logits(x, u, temperature=t)
        assert torch.equal(x.gather(1, ids[:, None])[:, 0], best)


def test_rows_past_a_launch_dimension_have_losses_and_gradients():
    """Two logits and one entry: -log p of it, and p less 1 there. In units of 2^-24: the difference d of the logits is
    rounded (|d|), so are the exponential's argument (|d| e^-|d| each for log2 e and the product, under 1 together) and
    itself (2), the sum (1 of at most 2), its logarithm (2 of at most 0.7) and the loss's two additions (|loss| each): under
    8 + 3 |loss|. A probability takes the exponential's and the sum's errors: under 16, and half a step of 1."""
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(ROWS, 2, device=DEV, generator=g)
    ids = torch.randint(0, 2, (ROWS, 1), device=DEV, generator=g, dtype=torch.int32)
    values = torch.zeros(ROWS, 1, device=DEV)
    p = torch.softmax(x.double(), 1)
    want = -p.gather(1, ids.long())[:, 0].log()
    tol = 2.0 ** -24 * (8 + 3 * want)
    p.scatter_add_(1, ids.long(), torch.full_like(p[:, :1], -1.0))
    loss, grad = sl.distill_loss_and_grad(x, values, ids, reduction="none")
    assert bool(((loss.double() - want).abs() <= tol).all())
    assert float((grad.double() - p).abs().max()) <= 17 * 2.0 ** -24
    del grad
    x.requires_grad_()
    mean = sl.distill_loss(x, values, ids)
    mean.backward()
    mean = mean.detach()
    # the mean's own rounding beside its terms'
    assert abs(float(mean) - float(want.mean())) <= float(tol.mean()) + 2.0 ** -24 * float(want.mean())
    # the share of a row (1 / N, twice rounded) before the probabilities', in units of it
    assert float((x.grad.double() * ROWS - p).abs().max()) <= 20 * 2.0 ** -24


@pytest.mark.parametrize("N", [1, 1023, 1025, 16384, 16385, 70001])
@pytest.mark.parametrize("first", [True, False])
def test_means_over_many_rows_count_the_rows(N, first):
    """Equal logits, where every row that counts has a loss of log 8 at one entry: the mean is that, whichever rows
    have nothing, and the gradient's sum of absolute values over a row is 2 (1 - 1/8) over the count. `first`: the
    entry is the first one or the last of 70."""
    g = torch.Generator(device=DEV).manual_seed(N)
    x = torch.zeros(N, 8, device=DEV, requires_grad=True)
    ids = torch.full((N, 70), -1, device=DEV)
    some = torch.rand(N, device=DEV, generator=g) < 0.6
    some[N // 2] = True
    ids[some, 0 if first else 69] = 3
    values = torch.zeros(N, 70, device=DEV)
    labels = torch.full((N,), -100, device=DEV)
    labels[::5] = 3   # of rows with and without entries
    count = int((some | (labels == 3)).sum())
    loss = sl.distill_loss(x, values, ids, labels, alpha=0.5)
    loss.backward()
    loss = loss.detach()
    terms = (some.double() + (labels == 3).double()).sum().item() * 0.5
    want = terms * 2.0794415416798357 / count
    # log 8 takes the logarithm of an exact sum (2 units of 2^-24), its half is exact, a row adds two, the mean one
    tol = 5 * 2.0 ** -24 * max(want, 1.0) * 2.1
    assert abs(float(loss) - want) <= tol
    both, grad = sl.distill_loss_and_grad(x, values, ids, labels, alpha=0.5)
    assert abs(float(both) - want) <= tol
    rows = (some.double() + (labels == 3).double()) * 0.5 * 1.75 / count
    for got in (x.grad, grad):
        # 1/8 is exact; the share 1 / count and its products round three times, the two tokens' sums once each
        assert bool(((got.double().abs().sum(1) - rows).abs() <= 8 * 2.0 ** -24 * rows).all())


@pytest.mark.parametrize("K", [1, 2, 3, 16, 33, 64, 255, 256, 1000, 1024])
@pytest.mark.parametrize("N,V", [(3, 2000), (600, 90), (600, 1500), (520, 5003), (2, 9000)])
def test_entries_that_name_the_same_tokens(N, V, K):
    """Tokens named by many entries, by all of them, by two far apart, some by the label too: each has the sum of its
    entries' probabilities. Ids are int32 for odd K."""
    g = torch.Generator(device=DEV).manual_seed(K)
    x = 2 * torch.randn(N, V, device=DEV, generator=g)
    values = torch.randn(N, K, device=DEV, generator=g)
    few = torch.randint(0, V, (N, 1), device=DEV, generator=g)
    ids = torch.randint(0, V, (N, K), device=DEV, generator=g)
    ids[::4] = (few + 7 * torch.randint(0, 5, (N, K), device=DEV, generator=g))[::4] % V   # of five tokens
    ids[1::4] = few[1::4]                                                                   # of one
    ids[2::4, -1] = ids[2::4, 0]
    ids[:, K // 2] = torch.where(torch.rand(N, device=DEV, generator=g) < 0.3, -1, ids[:, K // 2])
    labels = torch.where(torch.rand(N, device=DEV, generator=g) < 0.5, ids[:, 0], few[:, 0])
    if K % 2:
        ids = ids.int()
    for lab in (None, labels):
        want = orc.distill(x, values, ids, lab, 2.0, 0.5, "sum")
        orc.check_distill(*sl.distill_loss_and_grad(x, values, ids, lab, temperature=2.0, reduction="sum"), want)
        xg = x.clone().requires_grad_()
        loss = sl.distill_loss(xg, values, ids, lab, temperature=2.0, reduction="sum")
        loss.backward()
        orc.check_distill(loss.detach(), xg.grad, want)


@pytest.mark.parametrize("groups", [128, 256, 512, 1024, 2048, 4096])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_at_the_sizes_where_threads_change(groups, dtype):
    """Rows that fill a form's registers, and one logit more or less: listed and drawn as the definitions do, and the same
    among many rows, which other forms may take."""
    unit = 16 // torch.tensor([], dtype=dtype).element_size()
    g = torch.Generator(device=DEV).manual_seed(groups)
    for V in (groups * unit - 1, groups * unit, groups * unit + 1):
        x = (3 * torch.randn(300, V, device=DEV, generator=g)).to(dtype)
        x[0] = x[0].round()
        x[1, V // 3:] = -float("inf")
        few = x[:8]
        for k in (1, 24, 25, 48, 49, 96, 97, 160, 161):
            values, ids = sl.top_logits(x, k)
            v, i = orc.top(few, k)
            assert torch.equal(values[:8].cpu().to(orc.F64), v) and torch.equal(ids[:8].cpu(), i), (V, k)
        u = torch.rand(300, device=DEV, generator=g)
        for limits in ((1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 70, 0.8, 0.01), (1.0, 0, 1.0, 0.05),
                       (1.0, 300, 0.95, 0.0)):
            got = sl.sample_logits(few, u[:8], *limits)
            assert torch.equal(got.cpu(), orc.sample(few, u[:8].cpu(), *limits)), (V, limits)
            all_rows = sl.sample_logits(x, u, *limits)
            parts = [sl.sample_logits(x[a:a + 60], u[a:a + 60], *limits) for a in range(0, 300, 60)]
            assert torch.equal(all_rows, torch.cat(parts)) and torch.equal(all_rows[:8], got), (V, limits)


def test_calls_of_two_threads_at_once():
    """Two host threads, a stream each, call everything on inputs of their own; each has what one thread alone gets."""
    def work(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        out = []
        for N, V in ((700, 300), (9, 40000), (600, 5000)):
            x = torch.randn(N, V, device=DEV, generator=g)
            values, ids = sl.top_logits(x, 20)
            xg = x.flip(0).requires_grad_()
            loss = sl.distill_loss(xg, values, ids, temperature=2.0)
            loss.backward()
            out += [values, ids, loss.detach(), xg.grad, *sl.distill_loss_and_grad(x, values, ids, ids[:, 0]),
                    sl.sample_logits(x, torch.rand(N, device=DEV, generator=g), top_p=0.9)]
        return out

    def on_a_stream(seed, results):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            results[seed] = [work(seed) for _ in range(5)]
        stream.synchronize()

    alone, together = {}, {}
    for seed in (1, 2):
        on_a_stream(seed, alone)
    threads = [threading.Thread(target=on_a_stream, args=(seed, together)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in (1, 2):
        for got in together[seed]:
            assert all(torch.equal(a, b) for a, b in zip(got, alone[seed][0]))


def test_limits_as_numbers_of_any_library():
    x = torch.randn(5, 300, device=DEV)
    u = torch.rand(5, device=DEV)
    want = sl.sample_logits(x, u, temperature=2, top_k=40, top_p=0.5, min_p=0.25)
    assert torch.equal(want.cpu(), orc.sample(x, u.cpu(), 2.0, 40, 0.5, 0.25))
    for number in (np.float32, np.float64):
        assert torch.equal(sl.sample_logits(x, u, number(2), np.int32(40), number(0.5), number(0.25)), want)
    assert torch.equal(sl.sample_logits(x, u, np.int64(2), 40.0, 0.5, 0.25), want)
