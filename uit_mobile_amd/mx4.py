"""Microscaled 4-bit matrices (OCP MXFP4) and the linear layer on them: HIP kernels of libuitk.so (csrc/mx4.hip).

`quantize(x)`      -> `Mx4Tensor`: 32 consecutive elements of the last dimension share a power-of-two scale (8 bits), an element is one of
                     +-{0, .5, 1, 1.5, 2, 3, 4, 6} times it: 4.25 bits an element.  A block holding an infinity or a NaN is NaN as a whole.
`Mx4Tensor.dequantize()`  the values the codes stand for
`linear(x, w)`     = residual + act(Q(x) @ W.T + bias) on the 4-bit matrix pipe; the sums are fp32, the output is rounded once.  `x` a tensor
                     (rounded to 4 bits on the way in) or an `Mx4Tensor`; `w` an `Mx4Tensor`, made once from the weights with `quantize`.
                     The same call gives the same bits; a row among a different number of rows may be added in another order (fp32 rounding)

What `UITBase(precision='mx4')` runs its dense layers on (uit_mobile_amd/models/uit.py), there in one order whatever the batch.  CUDA tensors only, on the tensors' device and its
current stream; enqueue-only, safe inside a HIP graph capture.  No gradients: like the rest of this package these are inference operators,
and a call that autograd would have to record is refused.
"""
import functools
import math
import struct

import torch

from . import _lib

_TYPES = {torch.float32: _lib.T_F32, torch.float16: _lib.T_F16, torch.bfloat16: _lib.T_BF16}
_ACTS = {None: 0, "relu": 1, "gelu": 2}
_RECORD_BYTES, _MAX_ROWS, _MAX_K = 4096 + 256, 1 << 31, 1 << 20             # uitk_mx4_bytes, without the call
_LINEAR_ARGS = struct.Struct("6Q6q4i")                                      # uitk_mx4_linear_args

# A call for a single token is a few microseconds of GPU time, so what happens here before the launch is most of it: arguments travel as packed
# bytes, a tensor is copied or converted only where it has to be, and the device is switched only where it is another one.


def run(fn, device, *args):
    """Enqueue fn(*args, stream) on `device` and its current stream."""
    i = device.index
    stream = torch._C._cuda_getCurrentRawStream(i)
    if torch._C._cuda_getDevice() == i:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(i):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, fn.__name__)


# The caller's tensor has new contents: its version counter says so, as after any in-place operation -- a backward pass that saved the old contents
# refuses, and a model whose parameter it is packs its weights again.
written = torch.autograd.graph.increment_version


def check_tensor(t, name):
    """A CUDA tensor of a type these operators take that needs no gradient -> its uitk_type (shared with norms.py)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: uit_mobile_amd has no CPU path")
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: this is an inference operator (call it under torch.no_grad())")
    return code


def as_rows(t, K):
    """[..., K] -> (a tensor that holds its rows, their distance in elements): `t` itself where its strides allow, else a copy."""
    if K > 1 and t.is_contiguous():
        return t, K
    rows = t.numel() // K if K else 0
    v = t.reshape(rows, K)
    if K > 1 and v.stride(1) != 1 or rows > 1 and v.stride(0) < K:
        v = v.contiguous()
    v = v.resolve_neg()                                                     # (imag of a conjugate: rows of one element reach this without a copy)
    return v, (v.stride(0) if rows > 1 else K)


def span(t):
    """The addresses a tensor's elements lie between (rows of one buffer that interleave count as sharing it)."""
    lo = t.data_ptr()
    if t.is_contiguous() or not t.numel():
        return lo, lo + t.numel() * t.element_size()
    return lo, lo + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()


def overlaps(a, b):
    """Do two spans share memory?"""
    return a[0] < b[1] and b[0] < a[1]


def new(shape, dtype, like):
    """An empty tensor on like's device (new_empty costs half of torch.empty where the type is the same)."""
    return like.new_empty(shape) if like.dtype is dtype else torch.empty(shape, dtype=dtype, device=like.device)


def check_vector(t, name, n, device, keep):
    """A per-channel parameter: [n] on `device` -> the address of its values in float32 (0: None).  What had to be converted joins `keep`."""
    if t is None:
        return 0
    if (n > 1 and isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.get_device() == device.index and t.dim() == 1 and t.numel() == n
            and t.is_contiguous() and not (t.requires_grad and torch.is_grad_enabled())):
        return t.data_ptr()
    check_tensor(t, name)
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be [{n}], got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    keep.append(t.to(torch.float32).resolve_neg().contiguous())
    return keep[-1].data_ptr()


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(M, N, K, x_type):
    return _lib.load().uitk_mx4_linear_workspace(M, N, K, x_type)


def _packed_bytes(rows, K):
    if rows > _MAX_ROWS or not 1 <= K <= _MAX_K:
        raise ValueError(f"a packed 4-bit matrix of {rows} rows x {K} is out of range (rows <= 2^31, 1 <= K <= 2^20)")
    return (rows + 63) // 64 * ((K + 127) // 128) * _RECORD_BYTES


class Mx4Tensor:
    """A packed 4-bit matrix: `shape` is the logical shape (blocks run along the last dimension), `data` the packed bytes -- an opaque
    order made for the matrix pipe (csrc/mx4_dev.h)."""

    def __init__(self, data, shape):
        shape = torch.Size(shape)
        if not shape or min(shape) < 0:
            raise ValueError(f"a packed matrix has at least one dimension and none below zero, got {tuple(shape)}")
        need = _packed_bytes(math.prod(shape[:-1]), shape[-1])
        if (not isinstance(data, torch.Tensor) or not data.is_cuda or data.dtype is not torch.uint8 or data.dim() != 1 or not data.is_contiguous()
                or data.numel() != need or data.data_ptr() % 16):
            raise ValueError(f"data must be the {need} packed bytes of a {tuple(shape)} matrix: a contiguous, 16-byte aligned uint8 CUDA tensor")
        self.data, self.shape = data, shape

    @classmethod
    def empty(cls, shape, device, rows=None):
        q = cls.__new__(cls)
        q.shape = shape = torch.Size(shape)
        q.data = torch.empty(_packed_bytes(math.prod(shape[:-1]) if rows is None else rows, shape[-1]), dtype=torch.uint8, device=device)
        return q

    @property
    def device(self):
        return self.data.device

    @property
    def rows(self):
        return math.prod(self.shape[:-1])

    def numel(self):
        return math.prod(self.shape)

    def __repr__(self):
        return f"Mx4Tensor({tuple(self.shape)}, device='{self.device}')"

    def dequantize(self, dtype=torch.float32):
        """The values, in `dtype` (exact in float32 and bfloat16; float16 rounds where a block's scale is out of its range)."""
        if dtype not in _TYPES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        if out.numel():
            K = self.shape[-1]
            run(_lib.entry("uitk_mx4_dequantize"), out.device, self.data.data_ptr(), out.numel() // K, K, out.data_ptr(), _TYPES[dtype], K)
        return out


def quantize(x):
    """x [..., K] (float32 / float16 / bfloat16) -> Mx4Tensor of the same shape."""
    code = check_tensor(x, "x")
    shape, device = x.shape, x.device
    if not shape or shape[-1] < 1:
        raise ValueError(f"x must be [..., K] with K >= 1, got {tuple(shape)}")
    K = shape[-1]
    rows = x.numel() // K
    q = Mx4Tensor.empty(shape, device, rows)
    if rows:
        v, ld = as_rows(x, K)
        run(_lib.entry("uitk_mx4_quantize"), device, v.data_ptr(), code, rows, K, ld, q.data.data_ptr())
    return q


def linear(x, w, bias=None, act=None, residual=None, out_dtype=None, out=None):
    """residual + act(Q(x) @ w.T + bias): x [..., K] tensor or Mx4Tensor, w Mx4Tensor [N, K], bias [N], act None / 'relu' / 'gelu' (x Phi(x), by
    a fitted polynomial: off by less than 2^-21 max(1, |y|)), residual [..., N] of the output's type -> [..., N].

    out_dtype: float32 / float16 / bfloat16 (default: x's type, or the residual's; float32 for a packed x), or 'mx4': the output is an
    Mx4Tensor, the next layer's x (no residual then).  out: write there instead (a contiguous tensor of the output's shape and type;
    `out=residual` accumulates in place)."""
    packed = isinstance(x, Mx4Tensor)
    x_type = _lib.T_MX4 if packed else check_tensor(x, "x")
    if not isinstance(w, Mx4Tensor):
        raise TypeError("w must be an Mx4Tensor: quantize(weight) once")
    if len(w.shape) != 2:
        raise ValueError(f"w must be [N, K], got {tuple(w.shape)}")
    N, K = w.shape
    x_shape, device = x.shape, x.device
    if len(x_shape) < 1 or x_shape[-1] != K:
        raise ValueError(f"x {tuple(x_shape)} does not match w {tuple(w.shape)}")
    if w.device != device:
        raise ValueError(f"w is on {w.device}, x on {device}")
    if act not in _ACTS:
        raise ValueError(f"act must be None, 'relu' or 'gelu', got {act!r}")
    shape = x_shape[:-1] + (N,)
    M = x.numel() // K
    if residual is not None:
        check_tensor(residual, "residual")
    if out is not None:
        check_tensor(out, "out")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else residual.dtype if residual is not None else torch.float32 if packed else x.dtype
    to_mx4 = out_dtype == "mx4"
    if not to_mx4 and out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be float32, float16, bfloat16 or 'mx4', got {out_dtype}")
    keep = []
    b = check_vector(bias, "bias", N, device, keep)
    res, ldr = None, 0
    if residual is not None:
        if to_mx4:
            raise ValueError("a residual needs an output of 16 or 32 bits")
        if residual.shape != shape or residual.dtype != out_dtype or residual.device != device:
            raise ValueError(f"residual must be {tuple(shape)} {out_dtype} on {device}, got {tuple(residual.shape)} {residual.dtype} on {residual.device}")
        res, ldr = as_rows(residual, N)
    if out is not None:
        if to_mx4:
            raise ValueError("out is not supported for a 4-bit output")
        if out.shape != shape or out.dtype != out_dtype or out.device != device or not out.is_contiguous() or out.is_neg():
            raise ValueError(f"out must be a contiguous {tuple(shape)} {out_dtype} on {device}")
        mine = span(out)
        for name, t in (("x", x.data if packed else x), ("w", w.data), ("bias", bias)):
            if t is not None and overlaps(mine, span(t)):
                raise ValueError(f"out shares memory with {name}")
        if residual is not None and overlaps(mine, span(residual)) and not (out.data_ptr() == residual.data_ptr() and residual.is_contiguous()):
            raise ValueError("out shares memory with the residual without being the residual")
    if to_mx4:
        result = Mx4Tensor.empty(shape, device, M)
        dst, out_type = result.data, _lib.T_MX4
    else:
        result = dst = new(shape, out_dtype, w.data if packed else x) if out is None else out
        out_type = _TYPES[out_dtype]
    if M == 0:
        return result
    src, ldx = (x.data, 0) if packed else as_rows(x, K)
    need = _workspace_bytes(M, N, K, x_type)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    args = _LINEAR_ARGS.pack(src.data_ptr(), w.data.data_ptr(), b, 0 if res is None else res.data_ptr(), dst.data_ptr(), 0 if ws is None else ws.data_ptr(),
                             M, N, K, ldx, ldr, N, x_type, out_type, _ACTS[act], 0)
    run(_lib.packed("uitk_mx4_linear"), device, args)
    if out is not None:
        written(out)
    return result
