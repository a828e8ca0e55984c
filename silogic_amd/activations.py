"""Activations in 8 bits: what gate layers keep of their input between the
forward and the backward of a training step.

A sample's row is held as one byte per value with an offset and a step of its
own: ``lo = min x``, ``step = (max x - lo) / 255``, ``code = rint((x - lo) *
(255 / (max x - lo)))``, standing for ``lo + code * step`` (off by at most half
a step; rows of bits come back exactly). A row that holds an infinity or a NaN,
or whose range overflows fp32, comes back as NaN. The reference keeps fp32
(kernels/dense.py:60-75)."""
import torch

from . import ops


def pack_rows8(x):
    """``x [B, D]`` -> ``(codes, rows)``: ``codes [ceil(B/4), D, 4]`` uint8
    (byte ``v`` of ``[t, i]`` is sample ``4t + v``, input ``i``; 0 past the
    batch), ``rows [B, 2]`` fp32 offsets and steps. Other types than fp32 are
    converted first."""
    ops.require_gpu(x)
    if x.dim() != 2 or x.shape[1] < 1 or not x.dtype.is_floating_point:
        raise ValueError(f"pack_rows8: {x.dtype} {tuple(x.shape)}, floating [B, D] expected")
    codes, rows = ops.rows8_pack(ops._as_f32(x))
    return codes if codes.shape[1] == x.shape[1] else codes[:, :x.shape[1]], rows


def unpack_rows8(codes, rows):
    """The values ``[B, D]`` fp32 that :func:`pack_rows8`'s result stands for."""
    ops.require_gpu(codes, rows)
    ops.same_device("unpack_rows8", codes, rows)
    if codes.dtype != torch.uint8 or codes.dim() != 3 or codes.shape[2] != 4 or codes.shape[1] < 1:
        raise ValueError(f"unpack_rows8: codes {codes.dtype} {tuple(codes.shape)}")
    T, D, _ = codes.shape
    if rows.dtype != torch.float32 or rows.dim() != 2 or rows.shape[1] != 2 or (rows.shape[0] + 3) // 4 != T:
        raise ValueError(f"unpack_rows8: rows {rows.dtype} {tuple(rows.shape)} for {T} tiles of 4 samples")
    ld = (D + 3) // 4 * 4
    if codes.stride() != (4 * ld, 4, 1) or codes.data_ptr() % 16:   # not pack_rows8's own: into its layout
        whole = codes.new_zeros((T, ld, 4))
        whole[:, :D] = codes
        codes = whole
    return ops.rows8_unpack(codes, ops._c(rows), D)


def save_activations(model, bits=8):
    """Have every gate layer of ``model`` (:class:`LogicLayer` with arity-2
    gate16, walsh or multilinear nodes and at most 16 candidates) keep its
    input in ``bits`` bits for the backward: 8, or 32 to go back. Outputs do
    not change; gradients are taken at the 8-bit values. Returns how many
    layers were set; a model without one raises. LUT layers and conv blocks
    keep fp32: the LUT layers' backward has no form on codes, and a conv
    block's routes each pooled gradient by comparing the forward's exact
    values, which 8 bits would move at near-ties."""
    from .layers import LogicLayer
    if bits not in (8, 32):
        raise ValueError(f"save_activations: {bits} bits (8 or 32)")
    layers = [m for m in model.modules() if isinstance(m, LogicLayer) and m.takes_rows8()]
    if not layers:
        raise ValueError("save_activations: no arity-2 gate layer of at most 16 candidates")
    for m in layers:
        m.saved_bits = bits
    return len(layers)
