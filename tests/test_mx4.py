"""Packed 4-bit matrices and the linear layer on them (uit_mobile_amd/mx4.py, csrc/mx4.hip) against the definition in 64 bits.

Tolerances.  quantize: none, the rounding is exact arithmetic.  linear: products of 4-bit operands are exact in fp32, so an output differs
from the 64-bit sum only by the fp32 accumulation: the matrix instruction adds 64 products per step, at most two fp32 roundings or
truncations (2^-23 of the partial sums, which never exceed S = sum |x w|), and at most 16 partial sums are joined:
    |err| <= (2 ceil(K / 64) + 16) 2^-23 S
through an activation whose slope is at most 1.13 (GELU; its own evaluation in fp32: 2^-21 max(1, |y|)), plus half a step of the output's type."""
import ctypes
import math

import pytest
import torch

from uit_mobile_amd import _lib, mx4

gpu = pytest.mark.gpu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference_values(x):
    """The MXFP4 values of x (float64, CPU) by search over the code table: the nearest magnitude, the even code on a tie."""
    x = x.detach().cpu()
    K = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -K % 32)).unflatten(-1, (-1, 32))
    amax = v.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax).exponent - 1
    X = torch.where(amax > 0, e - 2, torch.full_like(e, -127)).clamp(min=-127)
    X = torch.where(torch.isfinite(amax), X, torch.zeros_like(X))
    unit = torch.ldexp(torch.ones_like(amax), X)
    y = (v / unit).abs().clamp(max=6.0)
    d = (y[..., None] - GRID).abs()
    best = d.amin(-1, keepdim=True)
    hits = d == best
    even = hits & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.int().argmax(-1), hits.int().argmax(-1))
    q = torch.copysign(GRID[code], v) * unit
    q = torch.where(torch.isfinite(v).all(-1, keepdim=True), q, torch.full_like(q, float("nan")))
    return q.flatten(-2)[..., :K]


def _rand(shape, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(dtype)


# ------------------------------------------------------------------------------------------------------------ without a GPU
def test_reference_on_known_blocks():
    x = torch.zeros(2, 32)
    x[0, :12] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.9, -0.26, 6.0])
    want = torch.tensor([4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, -0.5, 6.0], dtype=torch.float64)
    assert torch.equal(reference_values(x)[0, :12], want) and not reference_values(x)[1].any()


def test_refusals_before_any_launch():
    L = _lib.load()
    assert L.uitk_mx4_bytes(1, 1) == 4352 and L.uitk_mx4_bytes(65, 129) == 4 * 4352 and L.uitk_mx4_bytes(0, 5) == 0
    for rows, K in ((-1, 4), (1, 0), ((1 << 31) + 1, 4), (1, (1 << 20) + 1)):
        assert L.uitk_mx4_bytes(rows, K) == -1
    p = ctypes.c_void_p(1 << 20)                                             # never dereferenced: every call below is refused on the host
    bad = _lib.ERR_INVALID_ARG
    assert L.uitk_mx4_quantize(p, 3, 4, 32, 32, p, None) == bad              # type
    assert L.uitk_mx4_quantize(None, 0, 4, 32, 32, p, None) == bad
    assert L.uitk_mx4_quantize(p, 0, 4, 32, 31, p, None) == bad              # overlapping rows
    assert L.uitk_mx4_quantize(p, 0, 4, 32, 32, ctypes.c_void_p((1 << 20) + 8), None) == bad      # alignment
    assert L.uitk_mx4_quantize(p, 0, 4, 0, 32, p, None) == bad
    assert L.uitk_mx4_quantize(None, 0, 0, 32, 32, None, None) == 0          # zero rows
    assert L.uitk_mx4_dequantize(p, 4, 32, p, 3, 32, None) == bad
    assert L.uitk_mx4_dequantize(p, 4, 32, None, 0, 32, None) == bad
    assert L.uitk_mx4_linear(None, None) == bad

    def call(**kw):
        a = dict(x=1 << 20, w=1 << 21, out=1 << 22, M=4, N=8, K=32, ldx=32, ldo=8, x_type=0, out_type=0)
        a.update(kw)
        return L.uitk_mx4_linear(ctypes.byref(_lib.Mx4LinearArgs(**a)), None)
    for kw in (dict(x=None), dict(w=None), dict(out=None), dict(N=0), dict(K=0), dict(M=-1), dict(x_type=4), dict(out_type=-1), dict(act=3), dict(reserved=1), dict(ldx=31), dict(ldo=7),
               dict(w=(1 << 21) + 4), dict(residual=1 << 23, ldr=7), dict(residual=1 << 23, ldr=8, out_type=3), dict(x_type=3, x=(1 << 20) + 8),
               dict(out_type=3, out=(1 << 22) + 8)):
        assert call(**kw) == bad, kw
    for kw in (dict(x=(1 << 20) + 2), dict(out=(1 << 22) + 1, out_type=1), dict(bias=(1 << 23) + 2), dict(residual=(1 << 23) + 1, ldr=8, out_type=2)):
        assert call(**kw) == bad, kw
    big = dict(M=4096, N=4096, K=4096, ldx=4096, ldo=4096)                   # packs x first: needs the workspace it asked for
    assert L.uitk_mx4_linear_workspace(4096, 4096, 4096, 0) == L.uitk_mx4_bytes(4096, 4096) and L.uitk_mx4_linear_workspace(4096, 4096, 4096, 3) == 0
    assert call(**big) == bad and call(workspace=(1 << 24) + 8, **big) == bad
    assert L.uitk_mx4_linear_workspace(1, 64, 64, 0) == 0
    assert L.uitk_mx4_quantize(ctypes.c_void_p((1 << 20) + 1), 1, 4, 32, 32, p, None) == bad
    assert L.uitk_mx4_dequantize(p, 4, 32, ctypes.c_void_p((1 << 20) + 2), 0, 32, None) == bad
    assert call(M=0, x=None) == 0
    assert L.uitk_mx4_linear_workspace(4, 8, 32, 5) == -1 and L.uitk_mx4_linear_workspace(4, 0, 32, 0) == -1


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        mx4.quantize(torch.zeros(4, 32))
    with pytest.raises(TypeError):
        mx4.quantize([1.0])
    with pytest.raises(RuntimeError, match="CUDA"):
        mx4.linear(torch.zeros(4, 32), None)


# ------------------------------------------------------------------------------------------------------------------ quantize
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 31), (1, 768), (2, 33), (63, 64), (64, 128), (65, 129), (130, 1000), (252, 768)])
def test_quantize_is_the_definition(rows, K, dtype):
    x = _rand((rows, K), dtype, seed=rows * 1000 + K, spread=2.0)
    x[rows // 2] = 0.0
    got = mx4.quantize(x.cuda()).dequantize()
    assert torch.equal(got.cpu().double(), reference_values(x))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties_extremes_and_non_finite(dtype):
    fi = torch.finfo(dtype)
    x = torch.zeros(12, 64, dtype=dtype)
    ties = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.75, -0.25, -5.0, 6.0], dtype=torch.float32)
    for i, ex in enumerate((0, 5, -9)):
        x[i, :12] = (ties * 2.0 ** ex).to(dtype)
    x[3, :4] = torch.tensor([fi.max, -fi.max, fi.max / 3, 1.0]).to(dtype)
    x[4, :3] = torch.tensor([fi.tiny, fi.tiny / 2, -fi.tiny / 4]).to(dtype)               # subnormals of the type
    x[5, 40] = float("inf")                                                                # second block only
    x[6, 3] = float("nan")
    x[7, 3] = float("-inf")
    x[8] = -0.0
    x[9, :5] = torch.tensor([1.0, float("nan"), 3.0, float("inf"), 2.0])
    x[10, 32:] = 1.0
    got, want = mx4.quantize(x.cuda()).dequantize().cpu().double(), reference_values(x)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.isnan(got[5, 32:]).all() and not torch.isnan(got[5, :32]).any()


@gpu
def test_quantize_smallest_scales_of_float32():
    x = torch.zeros(4, 32)
    x[0, :4] = torch.tensor([2.0 ** -126, 1.5 * 2.0 ** -127, 2.0 ** -149, -(2.0 ** -128)])
    x[1, 0] = 2.0 ** -149
    x[2, :3] = torch.tensor([2.0 ** -125, 2.0 ** -128, 3 * 2.0 ** -129])
    x[3, :3] = torch.tensor([2.0 ** -124, 2.0 ** -127, 2.0 ** -128])
    assert torch.equal(mx4.quantize(x.cuda()).dequantize().cpu().double(), reference_values(x))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_rounds_once_and_strides_do_not_matter(dtype):
    x = _rand((70, 100), torch.float32, seed=5)
    want = reference_values(x).to(dtype)
    assert torch.equal(mx4.quantize(x.cuda()).dequantize(dtype).cpu(), want)
    wide = torch.full((70, 133), 9.0)
    wide[:, 3:103] = x
    for view in (wide.cuda()[:, 3:103], x.t().contiguous().cuda().t(), x.cuda().view(7, 10, 100)):
        assert torch.equal(mx4.quantize(view).dequantize(dtype).cpu().reshape(70, 100), want)
    assert torch.equal(mx4.quantize(x[:1].cuda().expand(5, 100)).dequantize(dtype).cpu(), want[:1].expand(5, 100))


@gpu
def test_quantize_empty_and_writes_nothing_behind_its_buffer():
    assert mx4.quantize(torch.zeros(0, 40, device="cuda")).dequantize().shape == (0, 40)
    L = _lib.load()
    x = _rand((65, 40), torch.float32).cuda()
    n = L.uitk_mx4_bytes(65, 40)
    buf = torch.full((n + 4096,), 171, dtype=torch.uint8, device="cuda")
    _lib.check(L.uitk_mx4_quantize(ctypes.c_void_p(x.data_ptr()), 0, 65, 40, 40, ctypes.c_void_p(buf.data_ptr()),
                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "quantize")
    out = torch.full((66, 50), 5.0, device="cuda")
    _lib.check(L.uitk_mx4_dequantize(ctypes.c_void_p(buf.data_ptr()), 65, 40, ctypes.c_void_p(out.data_ptr()), 0, 50,
                                     ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "dequantize")
    assert (buf[n:] == 171).all()
    assert (out[65] == 5.0).all() and (out[:, 40:] == 5.0).all() and torch.equal(out[:65, :40].cpu().double(), reference_values(x))


# -------------------------------------------------------------------------------------------------------------------- linear
def _act64(y, act):
    return y.clamp(min=0.0) if act == "relu" else y * torch.special.ndtr(y) if act == "gelu" else y


def check_linear(got, x, w, bias=None, act=None, residual=None):
    xq, wq = reference_values(x), reference_values(w)
    y = xq @ wq.T
    S = xq.abs() @ wq.abs().T
    if bias is not None:
        y = y + bias.cpu().double()
        S = S + bias.cpu().double().abs()
    K = x.shape[-1]
    tol = (2 * math.ceil(K / 64) + 16) * 2.0 ** -23 * S
    y = _act64(y, act)
    if act == "gelu":
        tol = 1.13 * tol + 2.0 ** -21 * y.abs().clamp(min=1.0)
    if residual is not None:
        y = y + residual.cpu().double()
        tol = tol + 2.0 ** -23 * y.abs()                                    # the fp32 sum with the residual
    fi = torch.finfo(got.dtype)
    tol = tol + y.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps
    err = (got.detach().cpu().double() - y).abs()
    assert got.shape == y.shape
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))


SHAPES = [(1, 1, 1), (1, 64, 128), (1, 2304, 768), (3, 65, 33), (13, 537, 1000), (31, 100, 4096), (33, 64, 64), (64, 129, 768), (65, 96, 100),
          (252, 768, 768), (300, 70, 257), (515, 640, 384)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_shapes(M, N, K, dtype):
    x, w = _rand((M, K), dtype, seed=M + N + K), _rand((N, K), torch.float32, seed=K + 1, spread=0.3) * K ** -0.5
    got = mx4.linear(x.cuda(), mx4.quantize(w.cuda()), out_dtype=torch.float32)
    check_linear(got, x, w)


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("M,N,K", [(5, 67, 96), (70, 132, 200), (257, 256, 160)])
def test_linear_epilogue(M, N, K, act, out_dtype):
    x, w = _rand((M, K), torch.bfloat16, seed=1), _rand((N, K), torch.float32, seed=2, spread=0.3) * K ** -0.5
    bias, res = _rand((N,), torch.float32, seed=3), _rand((M, N), out_dtype, seed=4)
    wq = mx4.quantize(w.cuda())
    check_linear(mx4.linear(x.cuda(), wq, bias=bias.cuda(), act=act, out_dtype=out_dtype), x, w, bias, act)
    check_linear(mx4.linear(x.cuda(), wq, bias=bias.cuda(), act=act, residual=res.cuda()), x, w, bias, act, res)
    acc = res.cuda()
    assert mx4.linear(x.cuda(), wq, act=act, residual=acc, out=acc) is acc
    check_linear(acc, x, w, None, act, res)


# what the tile kernels take: more than 128 tiles of 128 x 128; at least 512 of 256 x 128 and K >= 4096 (ragged edges in every direction)
TILES = [(1100, 1930, 130), (1024, 2304, 64), (3000, 920, 400), (16385, 513, 2049), (128 * 128, 1024, 2048), (8193, 2049, 4097), (8192, 2048, 4096)]


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("M,N,K", TILES)
def test_linear_many_rows(M, N, K, packed, out_dtype):
    """Against the 64-bit product of the operands' own values (that quantize is right is another test's business)."""
    x, w = _rand((M, K), torch.bfloat16, seed=M + N).cuda(), mx4.quantize((_rand((N, K), torch.float32, seed=K, spread=0.3) * K ** -0.5).cuda())
    bias, res = _rand((N,), torch.float32, seed=3).cuda(), _rand((M, N), out_dtype, seed=4).cuda()
    xq = mx4.quantize(x)
    a, b = xq.dequantize().double(), w.dequantize().double()
    S = a.abs() @ b.abs().T + bias.double().abs()
    tol = (2 * math.ceil(K / 64) + 16) * 2.0 ** -23 * S
    lin = a @ b.T + bias.double()
    fi = torch.finfo(out_dtype)
    for act, residual in ((None, None), ("relu", res), ("gelu", None)):
        got = mx4.linear(xq if packed else x, w, bias=bias, act=act, residual=residual, out_dtype=out_dtype).double()
        y, t = _act64(lin, act), tol
        if act == "gelu":
            t = 1.13 * tol + 2.0 ** -21 * y.abs().clamp(min=1.0)
        if residual is not None:
            y = y + residual.double()
            t = tol + 2.0 ** -23 * y.abs()
        assert ((got - y).abs() <= t + y.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps).all(), act


@gpu
@pytest.mark.parametrize("M,N,K", [(1100, 1930, 130), (16385, 1030, 4200), (700, 3000, 256)])
def test_linear_many_rows_to_four_bits_and_into_a_view(M, N, K):
    x, w = mx4.quantize(_rand((M, K), torch.float16, seed=M).cuda()), mx4.quantize((_rand((N, K), torch.float32, seed=K) * K ** -0.5).cuda())
    f = mx4.linear(x, w, act="relu", out_dtype=torch.float32)
    q = mx4.linear(x, w, act="relu", out_dtype="mx4")
    assert torch.equal(q.dequantize(), mx4.quantize(f).dequantize())
    w2 = mx4.quantize((_rand((40, N), torch.float32, seed=1) * N ** -0.5).cuda())
    assert torch.equal(mx4.linear(q, w2), mx4.linear(mx4.quantize(f), w2))
    L = _lib.load()
    buf = torch.full((M + 3, N + 8), 5.0, device="cuda")
    a = _lib.Mx4LinearArgs(x=x.data.data_ptr(), w=w.data.data_ptr(), out=buf.data_ptr(), M=M, N=N, K=K, ldo=N + 8, x_type=3, out_type=0, act=1)
    _lib.check(L.uitk_mx4_linear(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "linear")
    assert (buf[M:] == 5.0).all() and (buf[:, N:] == 5.0).all() and torch.equal(buf[:M, :N], f)


@gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_on_packed_activations_is_the_same_call(M, N, K):
    x, w = _rand((M, K), torch.bfloat16, seed=M), mx4.quantize((_rand((N, K), torch.float32, seed=9) * K ** -0.5).cuda())
    a, b = mx4.linear(x.cuda(), w, out_dtype=torch.float32), mx4.linear(mx4.quantize(x.cuda()), w)
    S = reference_values(x).abs() @ w.dequantize().cpu().double().abs().T
    assert ((a - b).abs().cpu().double() <= 2 * (2 * math.ceil(K / 64) + 16) * 2.0 ** -23 * S).all()


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 33, 64), (40, 70, 96), (200, 384, 256), (66, 129, 512)])
def test_linear_writes_the_next_layers_operand(M, N, K):
    """out_dtype 'mx4' = quantize of the float32 output of the same call, bit for bit."""
    x, w = _rand((M, K), torch.float16, seed=6), mx4.quantize((_rand((N, K), torch.float32, seed=7) * K ** -0.5).cuda())
    bias = _rand((N,), torch.float32, seed=8).cuda()
    f = mx4.linear(x.cuda(), w, bias=bias, act="gelu", out_dtype=torch.float32)
    q = mx4.linear(x.cuda(), w, bias=bias, act="gelu", out_dtype="mx4")
    assert isinstance(q, mx4.Mx4Tensor) and q.shape == (M, N)
    assert torch.equal(q.dequantize().cpu().double(), reference_values(f))
    # ... and is a good operand: the elements behind N add nothing, whatever was in the buffer before
    w2 = mx4.quantize((_rand((48, N), torch.float32, seed=10) * N ** -0.5).cuda())
    check_linear(mx4.linear(q, w2), reference_values(f), w2.dequantize())


@gpu
def test_linear_non_finite_stays_in_its_row():
    x, w = _rand((40, 256), torch.bfloat16, seed=1), _rand((70, 256), torch.float32, seed=2)
    x[7, 100] = float("inf")
    x[33, 0] = float("nan")
    wq = mx4.quantize(w.cuda())
    for xx in (x.cuda(), mx4.quantize(x.cuda())):
        for act in (None, "relu", "gelu"):
            got = mx4.linear(xx, wq, act=act, out_dtype=torch.float32).cpu()
            bad = torch.isnan(got).all(-1)
            assert bad[7] and bad[33] and bad.sum() == 2 and not torch.isnan(got[~bad]).any()


@gpu
def test_linear_leading_dimensions_views_and_empty():
    w = mx4.quantize(_rand((24, 96), torch.float32, seed=3).cuda())
    x = _rand((2, 5, 96), torch.float32, seed=4).cuda()
    want = mx4.linear(x.reshape(10, 96), w)
    assert torch.equal(mx4.linear(x, w).reshape(10, 24), want)
    assert torch.equal(mx4.linear(x[0, 0], w), want[0]) or torch.allclose(mx4.linear(x[0, 0], w), want[0], rtol=0, atol=1e-5)
    wide = torch.zeros(10, 131, device="cuda")
    wide[:, 5:101] = x.reshape(10, 96)
    assert torch.equal(mx4.linear(wide[:, 5:101], w), want)
    assert mx4.linear(x[:0], w).shape == (0, 5, 24)
    assert mx4.linear(x[:0], w, out_dtype="mx4").dequantize().shape == (0, 5, 24)


@gpu
def test_linear_leaves_its_surroundings_alone():
    M, N, K = 67, 70, 64
    L = _lib.load()
    x, w = _rand((M, K), torch.float32, seed=1).cuda(), mx4.quantize(_rand((N, K), torch.float32, seed=2).cuda())
    buf = torch.full((M + 3, N + 9), 5.0, device="cuda")
    a = _lib.Mx4LinearArgs(x=x.data_ptr(), w=w.data.data_ptr(), out=buf.data_ptr(), M=M, N=N, K=K, ldx=K, ldo=N + 9, x_type=0, out_type=0)
    _lib.check(L.uitk_mx4_linear(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "linear")
    assert (buf[M:] == 5.0).all() and (buf[:, N:] == 5.0).all()
    check_linear(buf[:M, :N], x, w.dequantize())


@gpu
def test_linear_same_bits_again_on_another_stream_and_in_a_graph():
    M, N, K = 300, 200, 500
    x, w = _rand((M, K), torch.bfloat16, seed=1).cuda(), mx4.quantize(_rand((N, K), torch.float32, seed=2).cuda())
    bias = _rand((N,), torch.float32, seed=3).cuda()
    call = lambda: mx4.linear(mx4.linear(x, w, bias=bias, act="gelu", out_dtype="mx4"), w2, out_dtype=torch.float32)
    w2 = mx4.quantize(_rand((96, N), torch.float32, seed=5).cuda())
    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = call()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for i in range(3):
        x.copy_(_rand((M, K), torch.bfloat16, seed=20 + i))
        g.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(replayed, call())


@gpu
def test_refusals():
    x, w = torch.zeros(4, 64, device="cuda"), mx4.quantize(torch.zeros(8, 64, device="cuda"))
    with pytest.raises(ValueError, match="match"):
        mx4.linear(x[:, :32], w)
    with pytest.raises(TypeError, match="Mx4Tensor"):
        mx4.linear(x, torch.zeros(8, 64, device="cuda"))
    with pytest.raises(ValueError, match="act"):
        mx4.linear(x, w, act="tanh")
    with pytest.raises(ValueError, match="bias"):
        mx4.linear(x, w, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        mx4.linear(x, w, residual=torch.zeros(4, 7, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        mx4.linear(x, w, residual=torch.zeros(4, 8, device="cuda"), out_dtype="mx4")
    with pytest.raises(TypeError):
        mx4.linear(x, w, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        mx4.quantize(torch.zeros(4, 64, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros((), device="cuda"))
    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros(3, 0, device="cuda"))
    big = torch.zeros(4, 200, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        mx4.linear(big.view(-1)[:256].view(4, 64), w, out=big.view(-1)[:32].view(4, 8))
    with pytest.raises(ValueError, match="shares memory"):
        mx4.linear(x, w, residual=big.view(-1)[4:36].view(4, 8), out=big.view(-1)[:32].view(4, 8))
    p = torch.zeros(4, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        mx4.quantize(p)
    with torch.no_grad():
        mx4.quantize(p)


@gpu
def test_packed_matrices_are_checked_where_they_are_made():
    q = mx4.quantize(_rand((70, 200), torch.float32).cuda())
    again = mx4.Mx4Tensor(q.data, (70, 200))
    assert torch.equal(again.dequantize(), q.dequantize()) and "70" in repr(again)
    assert torch.equal(mx4.Mx4Tensor(q.data, (7, 10, 200)).dequantize().view(70, 200), q.dequantize())
    for data, shape in ((q.data, (129, 200)), (q.data, (70, 257)), (q.data[1:], (70, 200)), (q.data.cpu(), (70, 200)), (q.data.float(), (70, 200)), (q.data, ()), (None, (70, 200))):
        with pytest.raises(ValueError):
            mx4.Mx4Tensor(data, shape)


@pytest.mark.parametrize("shape", [(), (-1, 32), (-64, -1, 32), (64, -32)])
def test_packed_shapes_without_a_meaning(shape):
    with pytest.raises(ValueError, match="at least one dimension and none below zero"):
        mx4.Mx4Tensor(None, shape)


@gpu
def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows of a large call are those of a small one."""
    K = 4096
    rows = (1 << 31) // K + 129
    x = torch.empty((rows, K), dtype=torch.bfloat16, device="cuda")
    x[:128] = 1.0
    tail = _rand((200, K), torch.bfloat16, seed=1).cuda()
    x[-200:] = tail
    q = mx4.quantize(x)
    assert torch.equal(q.dequantize(torch.bfloat16)[-200:], mx4.quantize(tail).dequantize(torch.bfloat16))
    w = mx4.quantize((_rand((40, K), torch.float32, seed=2) * K ** -0.5).cuda())
    got, want = mx4.linear(q, w)[-200:], mx4.linear(tail, w, out_dtype=torch.float32)
    S = mx4.quantize(tail).dequantize().double().abs() @ w.dequantize().double().abs().T
    assert ((got - want).abs().double() <= 2 * (2 * K / 64 + 16) * 2.0 ** -23 * S).all()
    del x, q, got
    M, N = 70000, 32768                                                      # an output of more than 2^31 elements
    x, w = _rand((M, 64), torch.bfloat16, seed=3).cuda(), mx4.quantize(_rand((N, 64), torch.float32, seed=4).cuda())
    y = mx4.linear(x, w)
    a, b = mx4.quantize(x[-100:]).dequantize().double(), w.dequantize().double()
    ref = a @ b.T
    assert ((y[-100:].double() - ref).abs() <= 18 * 2.0 ** -23 * (a.abs() @ b.abs().T) + ref.abs() * 2.0 ** -8 + 1e-38).all()


@gpu
@pytest.mark.parametrize("M,N,K", [(13, 300, 8192), (1500, 2000, 512), (8192, 2048, 4096)])
def test_every_kernel_under_capture_and_on_two_streams_at_once(M, N, K):
    xs = [_rand((M, K), torch.bfloat16, seed=i).cuda() for i in range(2)]
    w = mx4.quantize((_rand((N, K), torch.float32, seed=9) * K ** -0.5).cuda())
    want = [mx4.linear(x, w, act="gelu") for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = mx4.linear(xs[i], w, act="gelu")
    for i, s in enumerate(streams):
        torch.cuda.current_stream().wait_stream(s)
        got[i].record_stream(torch.cuda.current_stream())
        assert torch.equal(got[i], want[i])
    buf = xs[0].clone()
    graphs = []
    for _ in range(2):                                                       # two graphs of the same call, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = mx4.linear(buf, w, act="gelu")
        graphs.append((g, out))
    for i in (0, 1, 0, 1):
        buf.copy_(xs[i])
        for g, out in graphs:
            g.replay()
        assert torch.equal(mx4.linear(xs[1 - i], w, act="gelu"), want[1 - i])
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[i]) for _, out in graphs)


@gpu
def test_a_tensor_on_another_device_than_the_current_one_switches(monkeypatch):
    """One device here: the current one is made to look like another, so the call takes the switching path."""
    x, w = _rand((5, 64), torch.float32).cuda(), mx4.quantize(_rand((8, 64), torch.float32, seed=1).cuda())
    want = mx4.linear(x, w)
    seen = []
    real = torch.cuda.device
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", lambda i: (seen.append(i), real(i))[1])
    assert torch.equal(mx4.linear(x, w), want) and seen == [0]
