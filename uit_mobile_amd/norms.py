"""The seam between two transformer blocks as one HIP kernel (csrc/block_norm.hip): residual add, gate, residual scale and the norms around it.

    z  = post(y)                        norm behind the block (optional)
    r' = residual + gate * scale * z    gate per sequence or per token, scale per channel (LayerScale); both optional
    h  = pre(r')                        norm in front of the next block (optional)

What Block.forward of the reference does in separate operations between two linears (models/uit.py:245-248).  fp32 arithmetic whatever the
types, one rounding per output, h from the unrounded r'.  `UITBase(precision='mx4')` runs its blocks on it.  CUDA tensors only, enqueue-only
on the tensors' device and its current stream, no gradients (a call that autograd would have to record is refused).
"""
import struct

import torch

from . import _lib
from .mx4 import _TYPES, Mx4Tensor, as_rows, check_tensor, check_vector, new, overlaps, run, span, written

_ARGS = struct.Struct("10Q7q8if4x")                                          # uitk_block_norm_args
_KINDS = {"layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}


def _affine(norm, name, D, device, keep):
    """(gain, offset), each [D] or None -> their addresses"""
    try:
        w, b = norm
    except (TypeError, ValueError):
        raise TypeError(f"{name} must be a pair (weight, bias), each [{D}] or None") from None
    return check_vector(w, name, D, device, keep), check_vector(b, name, D, device, keep)


def block_norm(y, residual, *, post=None, gate=None, scale=None, pre=None, kind="layer", eps=1e-6, out_dtype=None, inplace=False):
    """-> (r', h).  residual [..., D]; y of its shape (its type may differ) or None: h = pre(residual) alone.

    post, pre: (weight, bias) of the norm, each [D] or None; None: no such norm (without `pre` h is None).  kind: 'layer' or 'rms', both norms.
    gate: y's shape (per token), or [B, D] / [B, 1, .., D] for y [B, ..., D] (per sequence).  scale: [D].  out_dtype of h: float32 / float16 / bfloat16
    (default: the residual's) or 'mx4' (an Mx4Tensor, for mx4.linear).  inplace: write r' into `residual`, whose rows must then be
    addressable in place (last dimension contiguous, leading ones flattening to one stride)."""
    r_type = check_tensor(residual, "residual")
    shape, device = residual.shape, residual.device
    if not shape or not 1 <= shape[-1] <= 16384:
        raise ValueError(f"residual must be [..., D] with 1 <= D <= 16384, got {tuple(shape)}")
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    D = shape[-1]
    rows = residual.numel() // D
    y_type, yv, ldy = 0, None, 0
    if y is None:
        if post is not None or gate is not None or scale is not None:
            raise ValueError("post, gate and scale need a block output y")
        if pre is None:
            raise ValueError("nothing to do: neither y nor pre")
    else:
        y_type = check_tensor(y, "y")
        if y.shape != shape or y.device != device:
            raise ValueError(f"y must have the residual's shape and device, got {tuple(y.shape)} on {y.device}")
        yv, ldy = as_rows(y, D)
    keep = []
    post_w, post_b = (0, 0) if post is None else _affine(post, "post", D, device, keep)
    pre_w, pre_b = (0, 0) if pre is None else _affine(pre, "pre", D, device, keep)
    s = 0 if scale is None else check_vector(scale, "scale", D, device, keep)
    g, ldg, gate_rows, gate_type = 0, 0, 1, 0
    if gate is not None:
        gate_type = check_tensor(gate, "gate")
        if gate.device != device:
            raise ValueError(f"gate is on {gate.device}, not on {device}")
        gs = gate.shape
        if gs != shape:
            if len(shape) < 3 or not (gs[0] == shape[0] and gs[-1] == D and gate.numel() == gs[0] * D and len(gs) in (2, len(shape))):
                raise ValueError(f"gate must be {tuple(shape)} (per token) or {(shape[0], D)} for a y of three or more dimensions (per sequence), got {tuple(gs)}")
            gate_rows = max(1, rows // max(1, shape[0]))
        gv, ldg = as_rows(gate, D)
        keep.append(gv)
        g = gv.data_ptr()
    if out_dtype is None:
        out_dtype = residual.dtype
    h, h_type, h_ptr = None, 0, 0
    if pre is not None:
        if out_dtype == "mx4":
            h, h_type = Mx4Tensor.empty(shape, device, rows), _lib.T_MX4
            h_ptr = h.data.data_ptr()
        elif out_dtype in _TYPES:
            h, h_type = new(shape, out_dtype, residual), _TYPES[out_dtype]
            h_ptr = h.data_ptr()
        else:
            raise TypeError(f"out_dtype must be float32, float16, bfloat16 or 'mx4', got {out_dtype}")
    r, ldr = as_rows(residual, D)
    if y is None:
        r_out, ro, ldro = residual, None, 0
    elif inplace:
        mine = span(residual)
        for name, t in (("gate", gate), ("scale", scale)) + tuple(("post", t) for t in post or ()) + tuple(("pre", t) for t in pre or ()):
            if t is not None and overlaps(mine, span(t)):
                raise ValueError(f"inplace: {name} shares memory with the residual")
        if overlaps(mine, span(y)) and not (residual.data_ptr() == y.data_ptr() and residual.stride() == y.stride() and residual.dtype == y.dtype):
            raise ValueError("inplace: y shares memory with the residual without being the residual")
        if rows and r.data_ptr() != residual.data_ptr():
            raise ValueError("inplace: the residual's rows cannot be addressed in place (its strides need a copy)")
        r_out, ro, ldro = residual, r, ldr
    else:
        r_out = ro = residual.new_empty(shape)
        ldro = D
    if rows == 0:
        return r_out, h
    args = _ARGS.pack(0 if yv is None else yv.data_ptr(), r.data_ptr(), 0 if ro is None else ro.data_ptr(), h_ptr, g, s, post_w, post_b, pre_w, pre_b,
                      rows, ldy, ldr, ldro, D, ldg, gate_rows, D, y_type, r_type, h_type, gate_type, _KINDS[kind], post is not None, pre is not None, eps)
    run(_lib.packed("uitk_block_norm"), device, args)
    if inplace and ro is not None:
        written(residual)
    return r_out, h
