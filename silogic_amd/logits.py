"""What comes after a network's logits: learning them from a teacher's and drawing tokens from them (no counterpart
in the reference, which trains on labels and answers with the largest class).

Logits are ``[..., V]`` in fp32, bf16 or fp16, of any strides; the kernels read rows of neighbouring values, and copy
others first. Everything is computed in 32 bits or more."""
import math

import torch
import torch.autograd.forward_ad as forward_ad

from . import ops


def _shape(what, name, t, shape):
    if t.shape != shape:
        raise ValueError(f"{what}: {name} {tuple(t.shape)}, {tuple(shape)} expected")


def _plain(t):
    return t.detach() if t.requires_grad else t


def _flat(t, dtype):
    t = _plain(t)
    return ops._c(t if t.dim() == 1 else t.reshape(-1), dtype)


def top_logits(logits, k):
    """The ``k`` largest logits of each row and their ids, ``(values, ids)`` ``[..., k]`` in the logits' type and
    int64: by value, equal values by the lower id. What a student keeps of its teacher (:func:`distill_loss`). A NaN
    or -inf is no token; past the tokens that are there values are -inf and ids -1. ``k`` is at most 1024, ``V``
    2^24. No gradient flows through it."""
    whole = ops.one_op("top_logits", logits)
    rows = ops.check_logits("top_logits", _plain(logits))
    if not 1 <= k <= min(rows.shape[1], 1024):
        raise ValueError(f"top_logits: {k} of {rows.shape[1]} logits (1 to 1024, and no more than there are)")
    if rows.get_device() < 0:
        ops.require_gpu(rows)
    if whole:
        values, ids = torch.ops.silogic_hip.top_logits(rows, k)
    else:
        values, ids = ops.top_logits(rows, k)
    if logits.dim() == 2:
        return values, ids
    return values.view(*logits.shape[:-1], k), ids.view(*logits.shape[:-1], k)


def _limit(name, v, lead, dtype, least, most):
    """A number in ``[least, most]``, or a tensor with one of each row."""
    if isinstance(v, torch.Tensor):
        if v.dtype.is_floating_point != dtype.is_floating_point or v.dtype in (torch.bool, torch.complex64, torch.complex128):
            raise TypeError(f"sample_logits: {name} of {v.dtype}")
        _shape("sample_logits", name, v, lead)
        return _flat(v, dtype)
    if not least <= v <= most:
        raise ValueError(f"sample_logits: {name} {v} outside [{least}, {most}]")
    if not isinstance(v, int if dtype == torch.int64 else (int, float)):   # another library's number
        if dtype == torch.int64 and v != int(v):
            raise TypeError(f"sample_logits: {name} {v} is no whole number")
        v = int(v) if dtype == torch.int64 else float(v)
    return v


def _sample(logits, u, temperature, top_k, top_p, min_p, mask):
    """The arguments as the kernel reads them."""
    lead = logits.shape[:-1]
    rows = ops.check_logits("sample_logits", _plain(logits))
    if rows.shape[1] > 1 << 24:
        raise ValueError(f"sample_logits: {rows.shape[1]} logits a row (at most 2^24)")
    if not u.dtype.is_floating_point:
        raise TypeError(f"sample_logits: u of {u.dtype}")
    _shape("sample_logits", "u", u, lead)
    f32 = torch.float32
    u = _flat(u, f32)
    t = _limit("temperature", temperature, lead, f32, 0.0, math.inf)
    k = _limit("top_k", top_k, lead, torch.int64, 0, (1 << 63) - 1)
    p = _limit("top_p", top_p, lead, f32, 0.0, 1.0)
    m = _limit("min_p", min_p, lead, f32, 0.0, 1.0)
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"sample_logits: mask of {mask.dtype} (bool)")
        if mask.shape != logits.shape:
            try:
                mask = mask.expand(logits.shape)
            except RuntimeError:
                raise ValueError(f"sample_logits: mask {tuple(mask.shape)} for logits {tuple(logits.shape)}") from None
        mask = mask.reshape(-1, rows.shape[1]) if mask.dim() != 2 else mask
        mask = mask if mask.stride(1) == 1 or mask.shape[1] == 1 else mask.contiguous()
    limits = (t, k, p, m)
    d = rows.get_device()
    # all in order (the usual call), or the check that says what is not
    there = d >= 0 and u.get_device() == d and (mask is None or mask.get_device() == d)
    for v in limits:
        there &= isinstance(v, (int, float)) or v.get_device() == d
    if not there:
        each = [v for v in limits if isinstance(v, torch.Tensor)]
        ops.require_gpu(rows, u, mask, *each)
        ops.same_device("sample_logits", rows, u, mask, *each)
    return rows, u, limits, mask


def sample_logits(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """A token id (int64) of each row of ``logits [..., V]`` from a random number ``u [...]`` in [0, 1).

    Tokens are taken by value, equal values by the lower id, with masses ``exp((logit - largest) / temperature)``.
    Kept are the first ``top_k`` (0: all); of these those before which lies less than ``top_p`` of their mass; of
    these those with a mass of at least ``min_p`` times the largest. The token drawn is the first whose running sum
    of kept masses passes ``u`` times their sum. ``temperature`` 0 takes the first token. Each limit is a number, or
    a tensor ``[...]`` with one of each row (in fp32; there a temperature that is not over 0 takes the first
    token, and limits out of their range act as their nearest bound). ``mask`` (bool, ``[V]`` to ``[..., V]``) is True for
    tokens that are allowed. A NaN or -inf is no token; a row without one gives -1.

    Masses are held as whole numbers of 2^-F of the largest, so that their sums are exact and the same draw comes from
    the same inputs on every call. F is at most 50 and 62 less the bits of V, or from 2^18 logits on of the row's own
    sum: a border between tokens is off by 2^-43 and V 2^-(F+1) largest masses, together 2^-27 of the sum at most. A
    ``u`` outside [0, 1) acts as its nearest bound."""
    whole = ops.one_op("sample_logits", logits, u, temperature, top_k, top_p, min_p, mask)
    rows, u, limits, mask = _sample(logits, u, temperature, top_k, top_p, min_p, mask)
    if whole:
        number = [0 if isinstance(v, torch.Tensor) else v for v in limits]
        ids = torch.ops.silogic_hip.sample_logits(rows, u, *(kind(v) for kind, v in zip((float, int, float, float), number)),
                                                  *(v if isinstance(v, torch.Tensor) else None for v in limits), mask)
    else:
        ids = ops.sample_logits(rows, u, *limits, mask)
    return ids if logits.dim() == 2 else ids.view(logits.shape[:-1])


def _distill(what, logits, values, ids, labels, temperature, alpha, reduction):
    """The arguments as the kernels read them."""
    lead = logits.shape[:-1]
    rows = ops.check_logits(what, logits)
    if values.dtype not in ops.TABLE_DTYPES or ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: values of {values.dtype} (fp32, bf16 or fp16), ids of {ids.dtype} (int32 or int64)")
    if values.dim() < 1 or not 1 <= values.shape[-1] <= 1024:
        raise ValueError(f"{what}: values {tuple(values.shape)}, [..., K] of 1 to 1024 expected")
    _shape(what, "values", values, (*lead, values.shape[-1]))
    _shape(what, "ids", ids, values.shape)
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"{what}: temperature {temperature} outside [1e-4, 1e4]")
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"{what}: alpha {alpha} outside [0, 1]")
    if reduction not in ops.REDUCTIONS:
        raise ValueError(f"{what}: reduction {reduction!r} (none, sum or mean)")
    if labels is not None:
        if labels.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{what}: labels of {labels.dtype} (int32 or int64)")
        _shape(what, "labels", labels, lead)
        if labels.dim() != 1:
            labels = labels.reshape(-1)
        labels = labels.contiguous()
    if values.dim() != 2:
        values, ids = values.reshape(-1, values.shape[-1]), ids.reshape(-1, values.shape[-1])
    d = rows.get_device()
    # all in order (the usual call), or the check that says what is not
    if not (d >= 0 and values.get_device() == d and ids.get_device() == d and (labels is None or labels.get_device() == d)):
        ops.require_gpu(rows, values, ids, labels)
        ops.same_device(what, rows, values, ids, labels)
    return (rows, values.contiguous(), ids.contiguous(), labels, float(temperature), float(alpha),
            ops.REDUCTIONS[reduction])


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, values, ids, labels, *how):
        loss, kept = ops.distill_fwd(rows, values, ids, labels, *how)
        ctx.save_for_backward(rows, values, ids, labels, kept)
        ctx.how = how
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        rows, values, ids, labels, kept = ctx.saved_tensors
        return ops.distill_bwd(rows, values, ids, labels, *ctx.how, kept, g), None, None, None, None, None, None


def distill_loss(logits, values, ids, labels=None, temperature=1.0, alpha=0.5, reduction="mean"):
    """Loss of a student's ``logits [..., V]`` against a teacher's largest ones, ``values`` and ``ids`` ``[..., K]``
    (:func:`top_logits`; ``K`` at most 1024, ids int32 or int64), and against ``labels [...]`` where they are given:

        (1 - alpha) T^2 KL(softmax(values / T) || softmax(logits / T)) + alpha cross_entropy(logits, labels)

    (the first term alone, without its factor, where not). The teacher's probabilities q are those of its entries
    among themselves, KL is the sum of q_j (log q_j - log p[ids_j]) over the entries: a token that two of them name
    gets both their probabilities, each with its own logarithm. An entry with an id outside 0..V-1 or a value of -inf
    is absent, so is a label outside 0..V-1. A term without an entry or a label, or with a factor of 0, counts 0, as
    does a row of -inf alone; ``mean`` is over the rows with an entry or a label.

    ``temperature`` lies in 1e-4 to 1e4. Over 4 a small first term is summed without cancellation; up to 4, and in the
    gradient, two 32-bit numbers are subtracted (the loss is off by some T^2 2^-21 then, a gradient by some T 2^-22 of
    the probabilities). Losses are fp32; the logits' gradient is in their type, rounded once, and the same bits on
    every call. The teacher gets no gradient, and there is no second derivative, none in forward mode and no
    ``torch.func`` transform."""
    whole = ops.one_op("distill_loss", logits, values, ids, labels)
    if not torch.compiler.is_compiling() and forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError("distill_loss: no derivative in forward mode")
    args = _distill("distill_loss", logits, values, ids, labels, temperature, alpha, reduction)
    if whole:
        loss = torch.ops.silogic_hip.distill_loss(*args)[0]
    elif ops._grad_path(logits):
        loss = _DistillFn.apply(*args)
    else:
        loss = ops.distill_fwd(*args)[0]
    return loss.view(logits.shape[:-1]) if reduction == "none" and logits.dim() != 2 else loss


def distill_loss_and_grad(logits, values, ids, labels=None, temperature=1.0, alpha=0.5, reduction="mean", scale=1.0):
    """:func:`distill_loss` and its gradient by the logits (in their shape and type) from one call, for
    ``logits.backward(grad)``: ``scale`` is the loss's own upstream gradient (a loss scale, or one over the number of
    batches that are accumulated). The logits are read once where a row fits a workgroup's registers."""
    if not math.isfinite(scale):
        raise ValueError(f"distill_loss_and_grad: scale {scale}")
    whole = ops.one_op("distill_loss_and_grad", logits, values, ids, labels)
    args = _distill("distill_loss_and_grad", logits.detach(), values, ids, labels, temperature, alpha, reduction)
    if whole:
        loss, grad = torch.ops.silogic_hip.distill_loss_grad(*args, float(scale))
    else:
        loss, grad = ops.distill_loss_grad(*args, float(scale))
    return (loss.view(logits.shape[:-1]) if reduction == "none" else loss), grad.view(logits.shape)
