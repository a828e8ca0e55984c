"""The operators on a network's logits, as they are timed: learning from a teacher's and drawing from them.

Three kinds of case, each a dict with ``op``:

``distill``  the loss of a student's logits against a teacher's largest ones (and against labels), and the
             gradient of the logits: through autograd, or with ``fused`` both from one call.
``top``      a teacher's ``K`` largest logits of each row with their token ids, as they are stored for a student.
``sample``   one token drawn from each row from a given random number, with a temperature and the limits
             top-k, top-p and min-p, one set for all rows or one for each.

With ``s`` a row of ``V`` logits, ``t_j`` at token ``i_j`` the teacher's entries and ``T`` the temperature:

distill: ``q = softmax(t / T)`` over the entries that are there (an id in ``0..V-1``, a value over -inf),
``soft = T^2 sum_j q_j (log q_j - log_softmax(s / T)[i_j])``, ``hard = -log_softmax(s)[label]``, the row's loss
``(1 - alpha) soft + alpha hard`` (``soft`` alone without labels). A term without an entry or without a label is
0. ``mean`` is over the rows that have either.

top: by value, equal values by the lower id.

sample: tokens in that same order, with masses ``exp((s - max s) / T)``. Kept are the first ``top_k``; of these
those before which lies less than ``top_p`` of their mass; of these those with a mass of at least ``min_p`` times
the largest. The token drawn is the first whose running sum of kept masses passes ``u`` times their sum. A
temperature of 0 takes the first token; a row without an allowed token gives -1.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MOST = 4096 * 32000   # logits of the largest case


def listed():
    return [
        # a character model's batch: launches and host calls
        dict(name="distill chars", op="distill", fused=False, dtype="float32", N=250, V=257, K=16, T=2.0, labels=False,
             reduction="mean"),
        # odd sizes in 16 bits, labels beside the teacher, a weight for each row
        dict(name="distill odd", op="distill", fused=False, dtype="bfloat16", N=333, V=4001, K=5, T=1.5, labels=True,
             reduction="none"),
        # few rows over a long vocabulary
        dict(name="distill long", op="distill", fused=False, dtype="float16", N=16, V=131071, K=64, T=1.0, labels=True,
             reduction="sum"),
        # a batch of words
        dict(name="distill words", op="distill", fused=False, dtype="float32", N=4096, V=32000, K=64, T=2.0,
             labels=False, reduction="mean"),
        # the same with labels, in 16 bits, loss and gradient from one call
        dict(name="distill words fused", op="distill", fused=True, dtype="bfloat16", N=4096, V=32000, K=64, T=2.0,
             labels=True, reduction="mean"),
        # a teacher of characters
        dict(name="top chars", op="top", dtype="float32", N=64, V=257, K=8),
        # a teacher's long rows, few of them
        dict(name="top long", op="top", dtype="float32", N=33, V=131071, K=100),
        # the targets of a batch of words
        dict(name="top words", op="top", dtype="bfloat16", N=4096, V=32000, K=64),
        # one token of one request
        dict(name="sample one", op="sample", rows="logits", limits="k", mask=False, dtype="float32", N=1, V=5000),
        # counts of a hard network's gates: many equal values
        dict(name="sample counts", op="sample", rows="counts", limits="p", mask=False, dtype="float32", N=4096, V=257),
        # requests with limits and allowed tokens of their own
        dict(name="sample serving", op="sample", rows="logits", limits="rows", mask=True, dtype="bfloat16", N=64,
             V=32000),
        # many rows of a long distribution, drawn from the most probable nine tenths
        dict(name="sample words", op="sample", rows="logits", limits="p", mask=False, dtype="float32", N=4096, V=32000),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["distill", "distill", "top", "sample", "sample"])
    V = _log(rng, 2, 160000)
    case = dict(op=op, dtype=rng.choice(["float32", "bfloat16", "float16"]), N=_log(rng, 1, max(1, min(8192, MOST // V))),
                V=V)
    if op == "distill":
        fused = rng.random() < 0.4
        case.update(fused=fused, K=_log(rng, 1, min(V, 256)), T=rng.choice([0.7, 1.0, 2.0, 4.0]),
                    labels=rng.random() < 0.5, reduction=rng.choice(["mean", "sum"] if fused else ["mean", "sum", "none"]))
    elif op == "top":
        case.update(K=_log(rng, 1, min(V, 256)))
    else:
        case.update(rows=rng.choice(["logits", "logits", "logits", "counts"]),
                    limits=rng.choice(["none", "k", "p", "m", "kp", "rows"]), mask=rng.random() < 0.3)
        if case["rows"] == "counts":
            case["dtype"] = "float32"
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rows(N, V, g):
    """Logits as a trained network gives them: a wide bulk, a few likely tokens above it, and how sure the
    network is differs from row to row."""
    s = torch.randn((N, V), generator=g, device=DEV).mul_(1.5 + 1.5 * torch.rand((N, 1), generator=g, device=DEV))
    n = min(V, 12)
    likely = (torch.randint(0, V, (N, 1), generator=g, device=DEV) + torch.arange(n, device=DEV) * (V // n)) % V
    return s.scatter_add_(1, likely, 4.0 + 6.0 * torch.rand((N, n), generator=g, device=DEV))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    N, V, dtype = case["N"], case["V"], DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "sample" and case["rows"] == "counts":
        # of 100 gates a class that each say yes half of the time, drawn at a temperature of a few counts
        s["logits"] = torch.round(50 + 5 * torch.randn((N, V), generator=g, device=DEV)).clamp_(0, 100)
    else:
        s["logits"] = _rows(N, V, g).to(dtype)
    if case["op"] == "distill":
        K = case["K"]
        teacher = s["logits"].float() + 2.0 * torch.randn((N, V), generator=g, device=DEV)
        values, ids = torch.topk(teacher, K, dim=1)
        # one row in sixteen is padding; one in eight has fewer entries than places for them
        padding = torch.rand((N, 1), generator=g, device=DEV) < 1 / 16
        short = torch.rand((N, 1), generator=g, device=DEV) < 1 / 8
        there = torch.arange(K, device=DEV) < torch.where(short, 1 + K // 2, K)
        s["ids"] = torch.where(there & ~padding, ids, torch.full_like(ids, -1))
        s["values"] = values.to(dtype)
        if case["labels"]:
            sure = torch.rand((N,), generator=g, device=DEV) < 0.7
            label = torch.where(sure, ids[:, 0], torch.randint(0, V, (N,), generator=g, device=DEV))
            s["label"] = torch.where(padding[:, 0], torch.full_like(label, -100), label)
        s["alpha"] = 0.25
        if case["reduction"] == "none":
            s["weight"] = torch.rand((N,), generator=g, device=DEV)
    elif case["op"] == "sample":
        s["u"] = torch.rand((N,), generator=g, device=DEV)
        s["T"], s["k"], s["p"], s["m"] = (4.0 if case["rows"] == "counts" else 0.8), 0, 1.0, 0.0
        limits = case["limits"]
        if "k" in limits:
            s["k"] = min(V, 50)
        if "p" in limits:
            s["p"] = 0.9
        if limits == "m":
            s["m"] = 0.05
        if limits == "rows":
            pick = torch.randint(0, 6, (N,), generator=g, device=DEV)
            rand = torch.rand((4, N), generator=g, device=DEV)
            s["T"] = torch.where(pick == 0, torch.zeros_like(rand[0]), 0.5 + rand[0])
            s["k"] = torch.where((pick == 1) | (pick == 4), (rand[1] * 100).long() + 1, torch.zeros_like(pick))
            s["p"] = torch.where((pick == 2) | (pick == 4), 0.5 + 0.5 * rand[2], torch.ones_like(rand[2]))
            s["m"] = torch.where(pick == 3, 0.2 * rand[3], torch.zeros_like(rand[3]))
        if case["mask"]:
            # allowed tokens of a grammar; some rows allow nothing
            share = torch.rand((N, 1), generator=g, device=DEV)
            s["allowed"] = torch.rand((N, V), generator=g, device=DEV) < torch.where(share < 0.05, 0.0, share)
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _plain_distill(s):
    x, V, T = s["logits"].float(), s["V"], s["T"]
    there = (s["ids"] >= 0) & (s["ids"] < V)
    at = torch.where(there, s["ids"], torch.zeros_like(s["ids"]))
    t = torch.where(there, s["values"].float() / T, torch.full_like(s["values"], -math.inf, dtype=torch.float32))
    some = there.any(1)
    top = torch.where(some, t.amax(1), torch.zeros_like(t[:, 0])).unsqueeze(1)
    e = torch.exp(t - top)
    total = e.sum(1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    q, logq = e / total, t - top - torch.log(total)
    most = x.amax(1, keepdim=True)

    def softmax(scale):
        """Probabilities and the log of their sum, of x * scale."""
        e = torch.exp((x - most) * scale)
        z = e.sum(1, keepdim=True)
        return e / z, (most * scale + torch.log(z))

    p, lse = softmax(1 / T)
    terms = torch.where(q > 0, q * (logq - x.gather(1, at) / T + lse), torch.zeros_like(q))
    ws = 1.0 - s["alpha"] if s["labels"] else 1.0
    loss = ws * T * T * terms.sum(1)
    grad = (p * some.unsqueeze(1)).scatter_add_(1, at, -q) * (ws * T)
    counts = some
    if s["labels"]:
        known = (s["label"] >= 0) & (s["label"] < V)
        y = torch.where(known, s["label"], torch.zeros_like(s["label"])).unsqueeze(1)
        p1, lse1 = softmax(1.0)
        w = s["alpha"] * known.unsqueeze(1)
        loss = loss + (w * (lse1 - x.gather(1, y)))[:, 0]
        grad += (p1 * w).scatter_add_(1, y, -w)
        counts = counts | known
    if s["reduction"] == "none":
        return {"loss": loss, "grad": (grad * s["weight"].unsqueeze(1)).to(s["logits"].dtype)}
    n = counts.sum().clamp(min=1) if s["reduction"] == "mean" else 1
    return {"loss": loss.sum() / n, "grad": (grad / n).to(s["logits"].dtype)}


def _plain_top(s):
    values, ids = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    return {"values": values[:, :s["K"]].contiguous(), "ids": ids[:, :s["K"]].contiguous()}


def _plain_sample(s):
    x = s["logits"].float()
    if s["mask"]:
        x = torch.where(s["allowed"], x, torch.full_like(x, -math.inf))
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    # a border between tokens is where a sum of thousands of masses passes u: in 64 bits
    col = lambda v: v.double().unsqueeze(1) if torch.is_tensor(v) else torch.full(  # noqa: E731
        (len(x), 1), float(v), device=DEV, dtype=torch.float64)
    T, k, p, m = (col(s[n]) for n in ("T", "k", "p", "m"))
    place = torch.arange(x.shape[1], device=DEV).unsqueeze(0)
    first = place == 0
    x = x.double()
    most = x[:, :1]
    mass = torch.exp((x - most) / torch.where(T > 0, T, torch.ones_like(T)))
    mass = torch.where((x > -math.inf) & ((T > 0) | first), mass, torch.zeros_like(mass))
    mass = torch.where((k <= 0) | (place < k), mass, torch.zeros_like(mass))
    run = mass.cumsum(1)
    keep = ((run - mass < p * run[:, -1:]) | (p >= 1) | first) & (mass >= m)
    mass = torch.where(keep, mass, torch.zeros_like(mass))
    run = mass.cumsum(1)
    passed = run > s["u"].double().unsqueeze(1) * run[:, -1:]
    at = passed.to(torch.uint8).argmax(1, keepdim=True)
    drawn = order.gather(1, at)[:, 0]
    return {"token": torch.where(most[:, 0] > -math.inf, drawn, torch.full_like(drawn, -1))}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(s):
    import silogic_amd as sl
    if s["op"] == "top":
        values, ids = sl.top_logits(s["logits"], s["K"])
        return {"values": values, "ids": ids}
    if s["op"] == "sample":
        return {"token": sl.sample_logits(s["logits"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["p"],
                                          min_p=s["m"], mask=s.get("allowed"))}
    args = dict(labels=s.get("label"), temperature=s["T"], alpha=s["alpha"], reduction=s["reduction"])
    if s["fused"]:
        loss, grad = sl.distill_loss_and_grad(s["logits"], s["values"], s["ids"], **args)
        return {"loss": loss, "grad": grad}
    x = s["logits"].detach().requires_grad_()
    loss = sl.distill_loss(x, s["values"], s["ids"], **args)
    return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, [x], s.get("weight"))[0]}


def run(state):
    if own:
        return _own(state)
    return {"distill": _plain_distill, "top": _plain_top, "sample": _plain_sample}[state["op"]](state)


def work(case):
    N, V, size = case["N"], case["V"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "distill":
        # logits in, their gradient out; the teacher's values and ids in. An exponential for each softmax,
        # its sum and the gradient's product
        n = 2 if case["labels"] else 1
        return dict(bytes=2.0 * N * V * size + N * case["K"] * (size + 8) + N * 12, flops=5.0 * n * N * V)
    if case["op"] == "top":
        return dict(bytes=1.0 * N * V * size + N * case["K"] * (size + 8), flops=1.0 * N * V)
    # logits and what is allowed in, tokens out. A comparison, an exponential and a sum
    return dict(bytes=1.0 * N * V * (size + (1 if case["mask"] else 0)) + N * 12, flops=4.0 * N * V)


# ---------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "sample":
        return None
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "top":
        return {"values": torch.topk(s["logits"].to(f64), case["K"], dim=1)[0], "ids": None}
    N, V, T = case["N"], case["V"], case["T"]
    soft_part = 1.0 - s["alpha"] if case["labels"] else 1.0
    loss = torch.zeros(N, device=DEV, dtype=f64)
    grad = torch.zeros((N, V), device=DEV, dtype=f64)
    counted = torch.zeros(N, device=DEV, dtype=torch.bool)
    part = max(1, (1 << 26) // V)
    for a in range(0, N, part):
        rows = slice(a, min(N, a + part))
        x, ids = s["logits"][rows].to(f64), s["ids"][rows]
        out = (ids < 0) | (ids >= V)
        # the teacher as a distribution over the whole vocabulary
        q = torch.log_softmax((s["values"][rows].to(f64) / T).masked_fill(out, -math.inf), 1).exp()
        has = ~out.all(1)
        q = torch.where(out | ~has.unsqueeze(1), torch.zeros_like(q), q)
        whole = torch.zeros_like(x).scatter_add_(1, ids.masked_fill(out, 0), q)
        logp = torch.log_softmax(x / T, 1)
        loss[rows] = soft_part * T * T * (torch.special.xlogy(whole, whole) - whole * logp).sum(1)
        grad[rows] = soft_part * T * (logp.exp() * has.unsqueeze(1) - whole)
        counted[rows] = has
        if case["labels"]:
            label = s["label"][rows]
            ok = (label >= 0) & (label < V)
            one = torch.zeros_like(x).scatter_(1, label.masked_fill(~ok, 0).unsqueeze(1), 1.0) * ok.unsqueeze(1)
            logp = torch.log_softmax(x, 1)
            loss[rows] -= s["alpha"] * (one * logp).sum(1)
            grad[rows] += s["alpha"] * (logp.exp() * ok.unsqueeze(1) - one)
            counted[rows] |= ok
    if case["reduction"] == "none":
        return {"loss": loss, "grad": grad * s["weight"].to(f64).unsqueeze(1)}
    n = max(1, int(counted.sum())) if case["reduction"] == "mean" else 1
    return {"loss": loss.sum() / n, "grad": grad / n}
