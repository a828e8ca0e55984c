"""Learnable encoders on the GPU: the thermometer of numbers
(silogic/encoders.py:12-49) and the bits of tokens."""
import torch
import torch.nn as nn

from . import _lib, ops
from .data import _encode


class _LearnedThermoFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, thresholds, scale):
        ctx.save_for_backward(x, thresholds)
        ctx.scale = scale
        F, T = thresholds.shape
        return _encode(x, thresholds, True, 2, T).to(torch.float32)

    @staticmethod
    def backward(ctx, g):
        x, thr = ctx.saved_tensors
        B, F = x.shape
        T = thr.shape[1]
        need_x, need_t = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        gx = torch.empty_like(x) if need_x else None
        gt = torch.empty_like(thr) if need_t else None
        ws = _lib.lib().slg_learned_thermo_bwd_workspace(B, F, T)
        work = torch.empty(max(ws, 1), device=x.device, dtype=torch.float32)
        _lib.call("slg_learned_thermo_bwd", ops._p(x), B, F, T, ops._p(thr), float(ctx.scale),
                  ops._p(ops._c(g, torch.float32)), ops._p(gx), ops._p(gt), ops._p(work), ws,
                  ops._stream(x))
        return gx, gt, None


class LearnedThermometerEncoder(nn.Module):
    """Thermometer encoder with learnable per-feature thresholds (arguments
    as silogic.encoders.LearnedThermometerEncoder): input ``[B, F]`` ->
    ``[B, F*bits]``, bit ``f*bits + i`` = ``x_f > t_{f,i}``. The soft forward
    returns the hard bits with the gradient of ``sigmoid((x - t) * scale)``
    (straight-through; the value is exact where the reference's
    ``hard + soft - soft.detach()`` carries fp32 rounding)."""

    def __init__(self, num_features, bits, init_lo=0.0, init_hi=1.0, scale=10.0):
        super().__init__()
        self.num_features = num_features
        self.bits = bits
        self.scale = scale
        t = torch.linspace(init_lo, init_hi, bits + 2)[1:-1]
        self.thresholds = nn.Parameter(t.repeat(num_features, 1))

    def forward(self, x):
        ops.require_gpu(x)
        return _LearnedThermoFn.apply(ops._as_f32(x), ops._c(self.thresholds, torch.float32),
                                      self.scale)

    @torch.no_grad()
    def forward_hard(self, x):
        ops.require_gpu(x)
        return _encode(ops._as_f32(x), ops._c(self.thresholds.detach(), torch.float32), True, 2,
                       self.bits)

    @torch.no_grad()
    def forward_packed(self, x, word_major=False):
        """The bits of :meth:`forward_hard` packed 64 samples per word:
        ``[F*bits, nw]`` (``word_major``: ``[nw, F*bits]``)."""
        ops.require_gpu(x)
        return _encode(ops._as_f32(x), ops._c(self.thresholds.detach(), torch.float32), True,
                       1 if word_major else 0, self.bits)


class _TokenFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, ste, pad):
        ctx.save_for_backward(ids, table)
        ctx.meta = (scale, pad)
        return ops.token_encode(ids, table, scale, ste, pad)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        ids, table = ctx.saved_tensors
        return None, ops.token_encode_bwd(ids, table, *ctx.meta, gy), None, None, None


class TokenEncoder(nn.Module):
    """Learned bits of discrete tokens (no counterpart in the reference, whose
    encoders take numbers): ids ``[B]`` or ``[B, L]`` (int32 or int64) ->
    ``[B, L*bits]``, feature ``l*bits + d`` of token ``l``.

    The soft forward is ``sigmoid(scale * weight[id])`` (``scale > 0``) in fp32, with ``ste``
    the hard bits ``weight[id] > 0`` under the same gradient (straight
    through); :meth:`forward_hard` and :meth:`forward_packed` are the hard
    bits. A token with id ``padding_idx``, or outside the table, is absent: its
    features are 0 and it adds to no gradient. ``weight [num_tokens, bits]``
    may be fp32, bf16 or fp16; its gradient sums each id's tokens in fp32 in
    one order (the same bits on every call)."""

    def __init__(self, num_tokens, bits, scale=1.0, ste=False, padding_idx=None):
        super().__init__()
        self._settle(torch.randn(num_tokens, bits), scale, ste, padding_idx)

    @classmethod
    def from_weight(cls, weight, scale=1.0, ste=False, padding_idx=None):
        """An encoder on ``weight [num_tokens, bits]`` itself (not a copy)."""
        enc = cls.__new__(cls)
        nn.Module.__init__(enc)
        enc._settle(weight, scale, ste, padding_idx)
        return enc

    def _settle(self, weight, scale, ste, padding_idx):
        self._check_weight(weight)
        V = weight.shape[0]
        if padding_idx is not None:
            if not -V <= padding_idx < V:
                raise ValueError(f"TokenEncoder: padding_idx {padding_idx} for {V} tokens")
            padding_idx %= V
        if not 0 < scale <= 2e38:   # the soft form falls where the bits rise; scale log2 e overflows
            raise ValueError(f"TokenEncoder: scale {scale} outside (0, 2e38]")
        self.scale, self.ste, self.padding_idx = float(scale), bool(ste), padding_idx
        self.weight = weight if isinstance(weight, nn.Parameter) else nn.Parameter(weight)

    @staticmethod
    def _check_weight(weight):
        if weight.dim() != 2 or weight.numel() == 0:
            raise ValueError(f"TokenEncoder: weight {tuple(weight.shape)}, [num_tokens, bits] expected")
        if weight.dtype not in ops.TABLE_DTYPES:
            raise TypeError(f"TokenEncoder: weight of {weight.dtype} (fp32, bf16 or fp16)")

    # the present weight's sizes: a weight may be replaced by one of others
    @property
    def num_tokens(self):
        return self.weight.shape[0]

    @property
    def bits(self):
        return self.weight.shape[1]

    def extra_repr(self):
        return (f"{self.num_tokens}, {self.bits}, scale={self.scale}, ste={self.ste}, "
                f"padding_idx={self.padding_idx}")

    @property
    def _pad(self):
        return -1 if self.padding_idx is None else self.padding_idx

    def _ids(self, ids, weight):
        """``ids`` as ``[B, L]``, on ``weight``'s device."""
        if ids.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"TokenEncoder: ids of {ids.dtype} (int32 or int64)")
        if ids.dim() not in (1, 2):
            raise ValueError(f"TokenEncoder: ids {tuple(ids.shape)}, [B] or [B, L] expected")
        d = ids.get_device()
        if d < 0 or d != weight.get_device():   # the check that says what is wrong
            ops.require_gpu(ids, weight)
            ops.same_device("TokenEncoder", ids, weight)
        return ops._c(ids if ids.dim() == 2 else ids.unsqueeze(1))

    def forward(self, ids):
        w = self.weight
        self._check_weight(w)
        ids = self._ids(ids, w)
        if torch.compiler.is_compiling():
            return torch.ops.silogic_hip.token_encode(ids, w, self.scale, self.ste, self._pad)
        w = ops._c(w)
        if not ops._grad_path(w):
            return ops.token_encode(ids, w, self.scale, self.ste, self._pad)
        return _TokenFn.apply(ids, w, self.scale, self.ste, self._pad)

    def _bit_table(self, weight):
        """Bit words of the weight, made once per version of it: the parameter
        itself, its storage, version counter and layout (writes through
        ``.data`` and replays of a graph that updates the weight count no
        version: ``derived.clear`` drops the words). Another stream than the
        one that made them waits for them. A captured call makes its own inside
        the graph, which then keeps them and reads the weight afresh on every
        replay; so does a call on a weight without a version (made in inference
        mode)."""
        if torch.cuda.is_current_stream_capturing() or weight.is_inference():
            self._check_weight(weight)
            return ops.token_bits(ops._c(weight.detach()))
        here = ops._stream(weight).value
        slot = self.__dict__.get("_derived_bits")
        # w: the weight as it was, whose memory stays taken by it
        if slot is not None:
            of, version, w, made_on, bits, done = slot
            if of is weight and version == weight._version and w.dtype == weight.dtype and w.is_set_to(weight):
                if made_on != here:
                    stream = torch.cuda.current_stream(weight.device)
                    stream.wait_event(done)
                    bits.record_stream(stream)
                return bits
        self._check_weight(weight)
        w = weight.detach()
        bits = ops.token_bits(ops._c(w))
        done = torch.cuda.current_stream(w.device).record_event()
        self._derived_bits = (weight, weight._version, w, here, bits, done)
        return bits

    def __getstate__(self):   # copies and pickles make their own bit table
        return {k: v for k, v in self.__dict__.items() if k != "_derived_bits"}

    def _hard(self, ids, layout):
        w = self.weight
        ids = self._ids(ids, w)
        return ops.token_encode_hard(ids, self._bit_table(w), w.shape[1], self._pad, layout)

    def forward_hard(self, ids):
        """uint8 bits ``[B, L*bits]``."""
        return self._hard(ids, 2)

    def forward_packed(self, ids, word_major=False):
        """The bits of :meth:`forward_hard` packed 64 samples per word:
        ``[L*bits, nw]`` (``word_major``: ``[nw, L*bits]``), the input of
        ``LogicNet.forward_hard_packed``."""
        return self._hard(ids, 1 if word_major else 0)
