"""Every kernel the product of 4-bit matrices can run on (csrc/mx4_plan.h chooses one by the sizes), each against the 64-bit product.

That a shape runs on the kernel it stands for is asserted from the library's own rule (mx4_plan.h, compiled here on the CPU), so that a moved
threshold cannot leave a kernel without a test.  Tolerances: those of test_mx4.py -- products of 4-bit operands are exact in fp32 and an
output differs from the 64-bit sum by the fp32 accumulation alone,
    |err| <= (2 ceil(K / 64) + 16) 2^-23 sum |x w|,
GELU by 2^-21 max(1, |y|) more (slope at most 1.13), the fp32 sum with a residual by 2^-23 |y|, the output's type by half a step."""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from uit_mobile_amd import _lib, mx4
from test_mx4 import DTYPES, _act64, _rand

gpu = pytest.mark.gpu
CSRC = Path(_lib.__file__).resolve().parent / "csrc"

# (M, N, K) -> the kernel, and whether a tensor is quantised in a launch of its own first
PLANS = {
    (1, 2304, 768): ("rows8", False),                # a single token
    (5, 1000, 4100): ("rows16", False),
    (1003, 537, 1000): ("rows64", False),            # 32 x 17 groups of 32 columns, 8 x 5 tiles; nothing is a multiple of anything
    (64, 16421, 130): ("rows64", False),             # the last group holds 37 of its 64 columns, the last record 2 of its 128 elements
    (40, 8000, 3900): ("rows8", True),
    (13, 8192, 8192): ("rows16", True),
    (128, 8200, 1500): ("rows64", True),
    (127, 16370, 260): ("rows64", True),             # 64 columns a group and a 4-bit output that ends inside a record
    (65, 16500, 200): ("tile128", True),
    (8193, 2049, 4097): ("tile256", True),
}
ROWS = [s for s, p in PLANS.items() if p[0].startswith("rows")]
ROWS64 = [s for s, p in PLANS.items() if p[0] == "rows64"]


# ------------------------------------------------------------------------------------------------------------ without a GPU
def test_the_shapes_run_on_the_kernels_they_stand_for(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "plan.cpp"
    src.write_text('#include "mx4_plan.h"\n#include <cstdio>\nusing namespace uitk;\n'
                   'int main() {\n    const char* name[] = {"rows8", "rows16", "rows64", "tile128", "tile256"};\n    long long M, N, K;\n'
                   '    while (scanf("%lld %lld %lld", &M, &N, &K) == 3) {\n        const Mx4Plan p = mx4_plan(M, N, K, false), q = mx4_plan(M, N, K, true);\n'
                   '        printf("%s %d %s %d\\n", name[p.kernel], p.quantize_first, name[q.kernel], q.quantize_first);\n    }\n}\n')
    exe = tmp_path / "plan"
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], input="".join("%d %d %d\n" % s for s in PLANS), text=True, capture_output=True, check=True).stdout.split("\n")
    for (shape, (kernel, first)), line in zip(PLANS.items(), out):
        assert line == f"{kernel} {int(first)} {kernel} 0", shape                  # (the same kernel for a packed x, which nobody quantises)
        need = _lib.load().uitk_mx4_linear_workspace(*shape, _lib.T_F16)            # ... and the built library says so too
        assert need == (_lib.load().uitk_mx4_bytes(shape[0], shape[2]) if first else 0), shape
    assert {p for p in PLANS.values()} >= {(k, f) for k in ("rows8", "rows16", "rows64") for f in (False, True)} | {("tile128", True), ("tile256", True)}


# ----------------------------------------------------------------------------------------------------------------------- GPU
def _operands(shape, dtype):
    M, N, K = shape
    x = _rand((M, K), dtype, seed=M + N).cuda()
    return x, mx4.quantize((_rand((N, K), torch.float32, seed=K, spread=0.3) * K ** -0.5).cuda()), _rand((N,), torch.float32, seed=3).cuda()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", list(PLANS))
def test_every_kernel_is_the_64_bit_product(shape, dtype):
    M, N, K = shape
    x, w, bias = _operands(shape, dtype)
    xq = mx4.quantize(x)
    a, b = xq.dequantize().double(), w.dequantize().double()
    lin = a @ b.T + bias.double()
    tol = (2 * math.ceil(K / 64) + 16) * 2.0 ** -23 * (a.abs() @ b.abs().T + bias.double().abs())
    for act, out_dtype, with_res in ((None, torch.float32, False), ("relu", torch.float16, True), ("gelu", torch.bfloat16, False), ("gelu", torch.float32, True)):
        res = _rand((M, N), out_dtype, seed=4).cuda() if with_res else None
        got = mx4.linear(x, w, bias=bias, act=act, residual=res, out_dtype=out_dtype)
        y, t = _act64(lin, act), tol
        if act == "gelu":
            t = 1.13 * tol + 2.0 ** -21 * y.abs().clamp(min=1.0)
        if res is not None:
            y = y + res.double()
            t = t + 2.0 ** -23 * y.abs()
        fi = torch.finfo(out_dtype)
        assert got.dtype == out_dtype and ((got.double() - y).abs() <= t + y.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps).all(), (act, out_dtype)
        # the same kernel on packed activations: the same products, added in the same order
        assert torch.equal(mx4.linear(xq, w, bias=bias, act=act, residual=res, out_dtype=out_dtype), got), (act, out_dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROWS)
def test_rows_kernels_write_the_next_layers_operand(shape, dtype):
    """A 4-bit output is the quantised float32 output, bit for bit, raw or packed x -- and a good operand: what lies behind N adds nothing."""
    x, w, bias = _operands(shape, dtype)
    f = mx4.linear(x, w, bias=bias, act="gelu", out_dtype=torch.float32)
    w2 = mx4.quantize((_rand((40, shape[1]), torch.float32, seed=1) * shape[1] ** -0.5).cuda())
    for xx in (x, mx4.quantize(x)):
        q = mx4.linear(xx, w, bias=bias, act="gelu", out_dtype="mx4")
        assert torch.equal(q.dequantize(), mx4.quantize(f).dequantize())
        assert torch.equal(mx4.linear(q, w2), mx4.linear(mx4.quantize(f), w2))


@gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", ROWS64)
def test_wide_rows_kernel_leaves_its_surroundings_alone(shape, packed):
    M, N, K = shape
    x, w, bias = _operands(shape, torch.float16)
    want = mx4.linear(x, w, bias=bias, act="relu", out_dtype=torch.float32)
    xx = mx4.quantize(x).data if packed else x
    L = _lib.load()
    need = L.uitk_mx4_linear_workspace(M, N, K, _lib.T_MX4 if packed else _lib.T_F16)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    buf = torch.full((M + 3, N + 9), 5.0, device="cuda")
    a = _lib.Mx4LinearArgs(x=xx.data_ptr(), w=w.data.data_ptr(), bias=bias.data_ptr(), out=buf.data_ptr(), workspace=ws.data_ptr(), M=M, N=N, K=K, ldx=K,
                           ldo=N + 9, x_type=_lib.T_MX4 if packed else _lib.T_F16, out_type=0, act=1)
    _lib.check(L.uitk_mx4_linear(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "linear")
    assert torch.equal(buf[:M, :N], want) and (buf[M:] == 5.0).all() and (buf[:, N:] == 5.0).all()


@gpu
@pytest.mark.parametrize("shape", ROWS64)
def test_wide_rows_kernel_keeps_non_finite_values_in_their_row(shape):
    x, w, _ = _operands(shape, torch.bfloat16)
    x[7, 100] = float("inf")
    x[33, 0] = float("nan")
    for xx in (x, mx4.quantize(x)):
        got = mx4.linear(xx, w, out_dtype=torch.float32)
        bad = torch.isnan(got).all(-1)
        assert bad[7] and bad[33] and int(bad.sum()) == 2 and not torch.isnan(got[~bad]).any()


@gpu
@pytest.mark.parametrize("shape", [s for s in ROWS if PLANS[s][1]] + [(1003, 537, 1000)])
def test_rows_kernels_in_a_graph_and_in_place(shape):
    """Captured with its own quantise launch and workspace, replayed on new inputs; a residual that is the output."""
    M, N, K = shape
    x, w, bias = _operands(shape, torch.bfloat16)
    res = _rand((M, N), torch.float32, seed=6).cuda()
    want = mx4.linear(x, w, bias=bias, residual=res)
    acc = res.clone()
    assert mx4.linear(x, w, bias=bias, residual=acc, out=acc) is acc and torch.equal(acc, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mx4.linear(x, w, bias=bias, residual=res)
    for i in range(3):
        x.copy_(_rand((M, K), torch.bfloat16, seed=30 + i))
        g.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, mx4.linear(x, w, bias=bias, residual=res))
