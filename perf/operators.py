"""The operators that a logic network trained on tokens adds to the gate layers, as they are timed.

Four kinds of case, each a dict with ``op``:

``layer8``  one training pass of an arity-2 gate layer that keeps its input in 8 bits between the
            forward and the backward: the output, and the gradients of the input, the connection
            logits and the node parameters.
``rows8``   the 8-bit form of a batch of activations and back: codes with an offset and a step per
            sample.
``tokens``  the token encoder (a learned row of soft bits per token id) forward, and with ``train``
            its table's gradient from an upstream one.
``packed``  the token encoder's hard bits, 64 samples a word, as the fused hard network takes them.

``own`` says whether :func:`run` calls the framework's operators or computes their plain form.

The 8-bit form of a row is defined with its 32-bit arithmetic: ``lo = min``, ``step = (max - lo) / 255``,
``code = rint((x - lo) * (255 / (max - lo)))``, and the value that a code stands for is
``lo + code * step``.
"""
import math

import torch

own = False

DEV = "cuda"
GATE16, WALSH, MULTILINEAR = 0, 1, 2
KINDS = {"gate16": GATE16, "walsh": WALSH, "multilinear": MULTILINEAR}
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

MOST_GATHERS = 4096 * 10000 * 16      # operand reads of the largest layer
MOST_VALUES = 4096 * 16380            # values of the largest batch of activations
MOST_TOKEN_VALUES = 4096 * 128 * 128  # values of the largest encoded batch


def listed():
    return [
        # the first layer of the smallest benchmark network: launches and host calls
        dict(name="layer8 gate16 small", op="layer8", node="gate16", B=256, IN=784, OUT=2000, K=8),
        # odd widths, a ragged batch and a candidate count without a compiled form of its own
        dict(name="layer8 walsh odd", op="layer8", node="walsh", B=333, IN=4001, OUT=2503, K=5),
        # a hidden layer of the widest gate16 network of the benchmark
        dict(name="layer8 gate16 wide", op="layer8", node="gate16", B=4096, IN=10000, OUT=10000, K=8),
        # a hidden layer of the widest walsh network, at half of its candidates
        dict(name="layer8 walsh wide", op="layer8", node="walsh", B=1024, IN=16380, OUT=16380, K=4),
        # activations of a few samples, at widths that no vector load divides
        dict(name="rows8 odd", op="rows8", B=37, D=10007),
        # activations of a whole batch of the widest network
        dict(name="rows8 large", op="rows8", B=4096, D=16380),
        # one token of one request
        dict(name="tokens one", op="tokens", train=False, ste=False, dtype="float32", B=1, L=1, V=256, D=16),
        # characters: a small vocabulary whose rows get many tokens each
        dict(name="tokens train chars", op="tokens", train=True, ste=True, dtype="float32", B=250, L=49, V=257,
             D=24),
        # a vocabulary of words in 16 bits, windows of text with padding
        dict(name="tokens train words", op="tokens", train=True, ste=False, dtype="bfloat16", B=1024, L=64,
             V=32000, D=64),
        # the largest batch, with a vocabulary of the size of its rows
        dict(name="tokens train large", op="tokens", train=True, ste=False, dtype="float32", B=4096, L=128,
             V=50001, D=128),
        # serving a few requests
        dict(name="packed small", op="packed", word_major=True, dtype="float32", B=64, L=16, V=5000, D=49),
        # bulk scoring: the rows that the per-layer circuit takes
        dict(name="packed large", op="packed", word_major=False, dtype="float32", B=65536, L=16, V=32000, D=64),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer8", "layer8", "rows8", "tokens", "tokens", "packed"])
    if op == "layer8":
        K = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 8, 11, 16])
        IN, OUT = _log(rng, 2, 16380), _log(rng, 1, 16380)
        top = min(4096, MOST_GATHERS // (2 * OUT * K), MOST_VALUES // max(IN, OUT))
        return dict(op=op, node=rng.choice(["gate16", "walsh", "multilinear"]), B=_log(rng, 1, max(1, top)),
                    IN=IN, OUT=OUT, K=K)
    if op == "rows8":
        D = _log(rng, 1, 65537)
        return dict(op=op, B=_log(rng, 1, max(1, min(8192, MOST_VALUES // D))), D=D)
    L, D, V = _log(rng, 1, 512), _log(rng, 1, 512), _log(rng, 2, 131072)
    if op == "tokens":
        top = max(1, min(8192, MOST_TOKEN_VALUES // (L * D)))
        return dict(op=op, train=rng.random() < 0.7, ste=rng.random() < 0.5,
                    dtype=rng.choice(["float32", "bfloat16", "float16"]), B=_log(rng, 1, top), L=L,
                    V=max(2, min(V, 3 * MOST_TOKEN_VALUES // (4 * D))), D=D)
    top = max(1, min(65536, MOST_TOKEN_VALUES // (L * D)))
    return dict(op=op, word_major=rng.random() < 0.5, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                B=_log(rng, 1, top), L=L, V=max(2, min(V, 3 * MOST_TOKEN_VALUES // (4 * D))), D=D)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _token_ids(case, g):
    """Token ids of windows of text: frequencies fall as one over the rank, ranks fall on ids at
    random, and a quarter of the windows end early (padding, id 0)."""
    B, L, V = case["B"], case["L"], case["V"]
    u = torch.rand((B, L), generator=g, device=DEV)
    rank = (torch.exp(u * math.log(V)).long() - 1).clamp_(0, V - 1)
    ids = torch.randperm(V, generator=g, device=DEV)[rank]
    length = (torch.rand((B, 1), generator=g, device=DEV) * 4 * L).long() + 1
    return torch.where(torch.arange(L, device=DEV) < length, ids, torch.zeros_like(ids))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=g, device=DEV)    # noqa: E731
    s = dict(case)
    if case["op"] == "layer8":
        B, IN, OUT, K = case["B"], case["IN"], case["OUT"], case["K"]
        s["x"] = rand(B, IN)
        s["cand"] = torch.randint(0, IN, (OUT, 2, K), generator=g, device=DEV, dtype=torch.int32)
        s["conn"] = randn(OUT, 2, K)
        s["raw"] = randn(OUT, 16 if case["node"] == "gate16" else 4)
        s["gy"] = randn(B, OUT)
        s["inv_tau"] = 0.5 if case["node"] == "walsh" else 1.0
    elif case["op"] == "rows8":
        # a layer's activations: each sample has a range of its own, some samples are bits
        x = rand(case["B"], case["D"])
        spread, at = rand(case["B"], 1), randn(case["B"], 1)
        s["x"] = torch.where(at > 1.0, (x > 0.5).float(), at * 0.1 + spread * x)
    else:
        s["ids"] = _token_ids(case, g)
        s["table"] = randn(case["V"], case["D"]).to(DTYPES[case["dtype"]])
        s["scale"] = 1.25
        if case.get("train"):
            s["gy"] = randn(case["B"], case["L"] * case["D"])
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
# the 16 two-input gates in the basis {1, a, b, ab}, by their truth tables
# f(a, b) = bit 3 - (2a + b) of the gate's number
def _basis(dtype):
    i = torch.arange(16, device=DEV)
    f00, f01, f10, f11 = (((i >> n) & 1).to(dtype) for n in (3, 2, 1, 0))
    return torch.stack([f00, f10 - f00, f01 - f00, f11 - f10 - f01 + f00], 1)


def _softmax(v):
    e = torch.exp(v - v.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _rows8(x):
    """Codes, offset and step of every row (module docstring)."""
    lo = x.amin(1, keepdim=True)
    span = x.amax(1, keepdim=True) - lo
    most = torch.full_like(span, 255.0)   # quotients of tensors: a number's would be a product with a reciprocal
    inv = torch.where(span > 0, most / span, torch.zeros_like(span))
    return torch.round((x - lo) * inv), lo, span / most


def _node(node, a, b, p, inv_tau):
    """y, and dy/dz where z is the node's value before its sigmoid (1 where it has none)."""
    z = p[:, 0] + p[:, 1] * a + p[:, 2] * b + p[:, 3] * (a * b)
    if node != "walsh":
        return z, torch.ones_like(z)
    y = _sigmoid(z * inv_tau)
    return y, y * (1 - y) * inv_tau


def _poly(node, raw):
    """The node's polynomial {1, a, b, ab} from its parameters, and what its chain rule needs."""
    if node == "gate16":
        q = _softmax(raw)
        return q @ _basis(raw.dtype), q
    if node == "walsh":
        t = raw
        return torch.stack([t[:, 0] - t[:, 1] - t[:, 2] + t[:, 3], 2 * (t[:, 1] - t[:, 3]),
                            2 * (t[:, 2] - t[:, 3]), 4 * t[:, 3]], 1), None
    q = _sigmoid(raw)   # values at (0,0), (1,0), (0,1), (1,1)
    return torch.stack([q[:, 0], q[:, 1] - q[:, 0], q[:, 2] - q[:, 0],
                        q[:, 3] - q[:, 1] - q[:, 2] + q[:, 0]], 1), q


def _poly_back(node, q, gp):
    """Gradient of the node's parameters from that of its polynomial."""
    g0, g1, g2, g3 = gp.unbind(1)
    if node == "gate16":
        gq = gp @ _basis(gp.dtype).t()
        return q * (gq - (q * gq).sum(1, keepdim=True))
    if node == "walsh":
        return torch.stack([g0, 2 * g1 - g0, 2 * g2 - g0, g0 - 2 * g1 - 2 * g2 + 4 * g3], 1)
    return torch.stack([g0 - g1 - g2 + g3, g1 - g3, g2 - g3, g3], 1) * q * (1 - q)


def _plain_layer8(s):
    x, gy, node = s["x"], s["gy"], s["node"]
    cand, w = s["cand"].long(), _softmax(s["conn"])
    p, q = _poly(node, s["raw"])
    a, b = (x[:, cand] * w).sum(-1).unbind(-1)
    y, _ = _node(node, a, b, p, s["inv_tau"])
    code, lo, step = _rows8(x)
    kept = (lo + code * step)[:, cand]                           # [B, OUT, 2, K]
    a, b = (kept * w).sum(-1).unbind(-1)
    gz = gy * _node(node, a, b, p, s["inv_tau"])[1]
    g = torch.stack([gz * (p[:, 1] + p[:, 3] * b), gz * (p[:, 2] + p[:, 3] * a)], -1)
    gw = (g.unsqueeze(-1) * kept).sum(0)
    gx = torch.zeros_like(x).index_add_(1, cand.reshape(-1),
                                        (g.unsqueeze(-1) * w).reshape(x.shape[0], -1))
    gp = torch.stack([gz.sum(0), (gz * a).sum(0), (gz * b).sum(0), (gz * a * b).sum(0)], 1)
    return {"y": y, "gx": gx, "gconn": w * (gw - (w * gw).sum(-1, keepdim=True)),
            "graw": _poly_back(node, q, gp)}


def _plain_tokens(s):
    ids, e = s["ids"], s["table"].float() * s["scale"]
    there = (ids != 0).unsqueeze(-1)
    y = ((e > 0).float() if s["ste"] else _sigmoid(e))[ids] * there
    out = {"y": y.reshape(ids.shape[0], -1)}
    if s["train"]:
        t = torch.exp(-e.abs())
        gy = s["gy"].view(*ids.shape, -1) * there
        # a frequent token's row sums 10^5 values: in 64 bits
        total = torch.zeros(e.shape, device=DEV, dtype=torch.float64).index_add_(
            0, ids.reshape(-1), gy.reshape(-1, e.shape[1]).double())
        out["gtable"] = (total * (s["scale"] * t / (1 + t) ** 2)).to(s["table"].dtype)
    return out


def _plain_packed(s):
    ids = s["ids"]
    B = ids.shape[0]
    bits = ((s["table"] > 0)[ids] & (ids != 0).unsqueeze(-1)).reshape(B, -1)
    rows = torch.zeros((-(-B // 64) * 64, bits.shape[1]), device=DEV, dtype=torch.int64)
    rows[:B] = bits
    words = (rows.view(-1, 64, bits.shape[1]) << torch.arange(64, device=DEV).view(1, 64, 1)).sum(1)
    return {"words": words if s["word_major"] else words.t().contiguous()}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(s):
    import silogic_amd as sl
    op = s["op"]
    if op == "layer8":
        x, conn, raw = (s[k].detach().requires_grad_() for k in ("x", "conn", "raw"))
        y = sl.ops.fc_layer8(x, s["cand"], conn, raw, KINDS[s["node"]], s["inv_tau"])
        gx, gconn, graw = torch.autograd.grad(y, [x, conn, raw], s["gy"])
        return {"y": y, "gx": gx, "gconn": gconn, "graw": graw}
    if op == "rows8":
        codes, rows = sl.pack_rows8(s["x"])
        return {"x": sl.unpack_rows8(codes, rows), "rows": rows}
    if "encoder" not in s:   # the module that a program keeps
        s["encoder"] = sl.TokenEncoder.from_weight(s["table"], scale=s["scale"], ste=s.get("ste", False),
                                                   padding_idx=0)
    enc = s["encoder"]
    if op == "packed":
        return {"words": enc.forward_packed(s["ids"], word_major=s["word_major"])}
    if not s["train"]:
        with torch.no_grad():
            return {"y": enc(s["ids"])}
    y = enc(s["ids"])
    return {"y": y, "gtable": torch.autograd.grad(y, [enc.weight], s["gy"])[0]}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "layer8":
        return _plain_layer8(state)
    if state["op"] == "rows8":
        code, lo, step = _rows8(state["x"])
        return {"x": lo + code * step, "rows": torch.cat([lo, step], 1)}
    return _plain_tokens(state) if state["op"] == "tokens" else _plain_packed(state)


def work(case):
    op = case["op"]
    if op == "layer8":
        B, IN, OUT, K = case["B"], case["IN"], case["OUT"], case["K"]
        per_out = 2 * K * 3 * 4 + (16 if case["node"] == "gate16" else 4) * 2 * 4
        # input and its gradient, output and its gradient; per output candidates, logits, parameters
        # and their gradients. Forward 2K products and sums, backward 2K for the operands again, 2K for
        # the weights' and 2K for the input's gradient, and about 40 for the node
        return dict(bytes=8.0 * B * (IN + OUT) + OUT * per_out, flops=float(B) * OUT * (16 * K + 40))
    if op == "rows8":
        # read x, write and read a byte each, write the values
        return dict(bytes=float(case["B"]) * case["D"] * 10 + case["B"] * 16, flops=6.0 * case["B"] * case["D"])
    B, L, V, D = case["B"], case["L"], case["V"], case["D"]
    N, size = B * L, DTYPES[case["dtype"]].itemsize
    rows = min(V, N) * D * size   # at most so many rows of the table are looked up
    if op == "packed":
        return dict(bytes=8.0 * N + rows + -(-B // 64) * 8 * L * D, flops=1.0 * N * D)
    if not case["train"]:
        return dict(bytes=8.0 * N + rows + 4.0 * N * D, flops=4.0 * N * D)
    return dict(bytes=8.0 * N + rows + 8.0 * N * D + V * D * size, flops=5.0 * N * D)


# ---------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------
def _exact_layer8(s, case):
    f64 = torch.float64
    B, IN, OUT, K = (case[k] for k in ("B", "IN", "OUT", "K"))
    node, tau_inv = case["node"], s["inv_tau"]
    c = s["conn"].to(f64)
    w = torch.exp(c - torch.logsumexp(c, -1, keepdim=True))
    raw = s["raw"].to(f64)
    # values of the node at (0,0), (0,1), (1,0), (1,1), and their derivative by each parameter
    corner = [(0, 0), (0, 1), (1, 0), (1, 1)]
    if node == "gate16":
        table = torch.tensor([[(i >> (3 - 2 * a - b)) & 1 for a, b in corner] for i in range(16)],
                             device=DEV, dtype=f64)
        p = torch.exp(raw - torch.logsumexp(raw, -1, keepdim=True))
        v = p @ table
        back = lambda gv: p * (gv @ table.t() - (gv * v).sum(1, keepdim=True))  # noqa: E731
    elif node == "walsh":
        signs = torch.tensor([[1, 2 * a - 1, 2 * b - 1, (2 * a - 1) * (2 * b - 1)] for a, b in corner],
                             device=DEV, dtype=f64)
        v = raw @ signs.t()
        back = lambda gv: gv @ signs  # noqa: E731
    else:
        order = [a + 2 * b for a, b in corner]
        q = torch.sigmoid(raw)
        v = q[:, order]
        back = lambda gv: (torch.zeros_like(q).index_copy_(  # noqa: E731
            1, torch.tensor(order, device=DEV), gv) * q * (1 - q))
    y = torch.empty((B, OUT), device=DEV, dtype=f64)
    gx = torch.zeros((B, IN), device=DEV, dtype=f64)
    gw = torch.zeros((OUT, 2, K), device=DEV, dtype=f64)
    gv = torch.zeros((OUT, 4), device=DEV, dtype=f64)
    flat = s["cand"].long().reshape(-1)
    code, lo, step = _rows8(s["x"])   # the format's codes (module docstring)
    part = max(1, min(B, (1 << 26) // (OUT * K)))
    for b0 in range(0, B, part):
        sl = slice(b0, min(B, b0 + part))
        full = s["x"][sl].to(f64)
        near = lo[sl].to(f64) + code[sl].to(f64) * step[sl].to(f64)

        def operands(x):
            got = x.index_select(1, flat).view(-1, OUT, 2, K)
            return got, (got * w).sum(-1)

        def blend(o):
            a, b = o[..., 0], o[..., 1]
            parts = torch.stack([(1 - a) * (1 - b), (1 - a) * b, a * (1 - b), a * b], -1)
            return a, b, parts, (parts * v).sum(-1)

        z = blend(operands(full)[1])[3]
        y[sl] = torch.sigmoid(z * tau_inv) if node == "walsh" else z
        got, o = operands(near)
        a, b, parts, z = blend(o)
        gz = s["gy"][sl].to(f64)
        if node == "walsh":
            h = torch.sigmoid(z * tau_inv)
            gz = gz * h * (1 - h) * tau_inv
        ga = gz * ((1 - b) * (v[:, 2] - v[:, 0]) + b * (v[:, 3] - v[:, 1]))
        gb = gz * ((1 - a) * (v[:, 1] - v[:, 0]) + a * (v[:, 3] - v[:, 2]))
        g = torch.stack([ga, gb], -1).unsqueeze(-1)
        gw += (g * got).sum(0)
        gx[sl].index_add_(1, flat, (g * w).reshape(g.shape[0], -1))
        gv += (gz.unsqueeze(-1) * parts).sum(0)
    return {"y": y, "gx": gx, "gconn": w * (gw - (w * gw).sum(-1, keepdim=True)), "graw": back(gv)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer8":
        return _exact_layer8(s, case)
    if case["op"] == "rows8":
        code, lo, step = _rows8(s["x"])   # the format's codes, offset and step
        lo, step = lo.double(), step.double()
        return {"x": lo + code.double() * step, "rows": torch.cat([lo, step], 1)}
    if case["op"] == "packed":
        return None
    ids, e = s["ids"], s["table"].double() * s["scale"]
    hard, soft = (e > 0).double(), torch.sigmoid(e)
    value = hard if case["ste"] else soft
    there = (ids != 0)
    y = torch.where(there.unsqueeze(-1), value[ids], torch.zeros((), device=DEV, dtype=torch.float64))
    out = {"y": y.reshape(ids.shape[0], -1)}
    if case["train"]:
        # rows of the tokens in order, summed by where each one's run ends
        flat = ids[there]
        order = torch.argsort(flat, stable=True)
        gy = s["gy"].view(*ids.shape, -1)[there].double()[order]
        count = torch.bincount(flat, minlength=case["V"])
        total = torch.segment_reduce(gy, "sum", lengths=count, axis=0, initial=0.0) if len(flat) else \
            torch.zeros_like(e)
        out["gtable"] = total * soft * torch.sigmoid(-e) * s["scale"]
    return out
