"""The seam between two transformer blocks as one HIP kernel (csrc/block_norm.hip): residual add, gate, residual scale and the norms around it.

    z  = post(y)                        norm behind the block (optional)
    r' = residual + gate * scale * z    gate per sequence or per token, scale per channel (LayerScale); both optional
    h  = pre(r')                        norm in front of the next block (optional)

What Block.forward of the reference does in separate operations between two linears (models/uit.py:244-247).  fp32 arithmetic whatever the
types, one rounding per output, h from the unrounded r'.  `UITBase(precision='mx4')` runs its blocks on it.  CUDA tensors only, enqueue-only
on the tensors' device and its current stream, no gradients (a call that autograd would have to record is refused).
"""
import ctypes

import torch

from . import _lib
from .mx4 import _TYPES, Mx4Tensor, _ptr, _stream, as_rows, check_tensor, check_vector, overlaps

_KINDS = {"layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}


def _affine(norm, name, D, device):
    """(gain, offset), each [D] or None -> (given, gain, offset)"""
    if norm is None:
        return False, None, None
    try:
        w, b = norm
    except (TypeError, ValueError):
        raise TypeError(f"{name} must be a pair (weight, bias), each [{D}] or None") from None
    return True, check_vector(w, f"{name} weight", D, device), check_vector(b, f"{name} bias", D, device)


def block_norm(y, residual, *, post=None, gate=None, scale=None, pre=None, kind="layer", eps=1e-6, out_dtype=None, inplace=False):
    """-> (r', h).  residual [..., D]; y of its shape (its type may differ) or None: h = pre(residual) alone.

    post, pre: (weight, bias) of the norm, each [D] or None; None: no such norm (without `pre` h is None).  kind: 'layer' or 'rms', both norms.
    gate: y's shape (per token), or [B, D] / [B, 1, .., D] for y [B, ..., D] (per sequence).  scale: [D].  out_dtype of h: float32 / float16 / bfloat16
    (default: the residual's) or 'mx4' (an Mx4Tensor, for mx4.linear).  inplace: write r' into `residual`, whose rows must then be
    addressable in place (last dimension contiguous, leading ones flattening to one stride)."""
    check_tensor(residual, "residual")
    if residual.dim() < 1 or not 1 <= residual.shape[-1] <= 16384:
        raise ValueError(f"residual must be [..., D] with 1 <= D <= 16384, got {tuple(residual.shape)}")
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    D, device, shape = residual.shape[-1], residual.device, residual.shape
    if y is None:
        if post is not None or gate is not None or scale is not None:
            raise ValueError("post, gate and scale need a block output y")
        if pre is None:
            raise ValueError("nothing to do: neither y nor pre")
    else:
        check_tensor(y, "y")
        if y.shape != shape or y.device != device:
            raise ValueError(f"y must have the residual's shape and device, got {tuple(y.shape)} on {y.device}")
    rows = residual.numel() // D
    has_post, post_w, post_b = _affine(post, "post", D, device)
    has_pre, pre_w, pre_b = _affine(pre, "pre", D, device)
    s = check_vector(scale, "scale", D, device)
    g, ldg, gate_rows = None, 0, 1
    if gate is not None:
        check_tensor(gate, "gate")
        if gate.device != device:
            raise ValueError(f"gate is on {gate.device}, not on {device}")
        if gate.shape == shape:
            gate_rows = 1
        elif len(shape) > 2 and gate.shape in ((shape[0], D), (shape[0],) + (1,) * (len(shape) - 2) + (D,)):
            gate_rows = max(1, rows // max(1, shape[0]))
        else:
            raise ValueError(f"gate must be {tuple(shape)} (per token) or {(shape[0], D)} for a y of three or more dimensions (per sequence), got {tuple(gate.shape)}")
        g, ldg = as_rows(gate.detach())
    if out_dtype is None:
        out_dtype = residual.dtype
    to_mx4 = out_dtype == "mx4"
    if has_pre and not to_mx4 and out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be float32, float16, bfloat16 or 'mx4', got {out_dtype}")
    if inplace and y is not None:
        for name, t in (("gate", gate), ("scale", scale), ("post weight", post_w), ("post bias", post_b), ("pre weight", pre_w), ("pre bias", pre_b)):
            if t is not None and overlaps(residual, t):
                raise ValueError(f"inplace: {name} shares memory with the residual")
        if overlaps(residual, y) and not (residual.data_ptr() == y.data_ptr() and residual.stride() == y.stride() and residual.dtype == y.dtype):
            raise ValueError("inplace: y shares memory with the residual without being the residual")
    r, ldr = as_rows(residual.detach())
    if y is None:
        r_out, ro, ldro = residual, None, 0
    elif inplace:
        if rows and r.data_ptr() != residual.data_ptr():
            raise ValueError("inplace: the residual's rows cannot be addressed in place (its strides need a copy)")
        r_out, ro, ldro = residual, r, ldr
    else:
        r_out = ro = torch.empty(shape, dtype=residual.dtype, device=device)
        ldro = D
    h = None if not has_pre else Mx4Tensor.empty(shape, device) if to_mx4 else torch.empty(shape, dtype=out_dtype, device=device)
    if rows == 0:
        return r_out, h
    yv, ldy = (None, 0) if y is None else as_rows(y.detach())
    a = _lib.BlockNormArgs(
        y=_ptr(yv), residual=_ptr(r), residual_out=_ptr(ro), h=None if h is None else _ptr(h.data if to_mx4 else h), gate=_ptr(g), scale=_ptr(s),
        post_w=_ptr(post_w), post_b=_ptr(post_b), pre_w=_ptr(pre_w), pre_b=_ptr(pre_b), rows=rows, ldy=ldy, ldr=ldr, ldro=ldro, ldh=D, ldg=ldg,
        gate_rows=gate_rows, D=D, y_type=0 if y is None else _TYPES[y.dtype], r_type=_TYPES[residual.dtype],
        h_type=_lib.T_MX4 if to_mx4 else _TYPES.get(out_dtype, 0), gate_type=0 if gate is None else _TYPES[gate.dtype], kind=_KINDS[kind],
        post=int(has_post), pre=int(has_pre), eps=float(eps))
    with torch.cuda.device(device):
        _lib.check(_lib.load().uitk_block_norm(ctypes.byref(a), _stream(device)), "uitk_block_norm")
    return r_out, h
