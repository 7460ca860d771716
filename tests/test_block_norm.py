"""The fused seam between two blocks (uit_mobile_amd/norms.py, csrc/block_norm.hip) against the formulas in 64 bits.

Tolerances.  r' = r + g s z: three roundings of fp32 on the product and one on the sum: 2^-22 (|r| + |g s z|), plus what a post norm adds; half a
step of the output's type.  A norm of D elements in fp32: mean and variance are sums of D terms added in chains of at most D / 64 + 16 steps, so
the normalised value is off by at most (D / 64 + 24) 2^-23 (|u| + |w|(1 + |mean| / deviation)), u the output -- the factor |mean| / deviation is the
cancellation in v - mean -- and an error d of the norm's input moves its output by at most 2 |w| max|d| / deviation (1 + |u|) for max|d| below the
deviation, the factor 2 for the mean and the deviation that move along."""
import ctypes

import pytest
import torch

from uit_mobile_amd import _lib, mx4, norms
from test_mx4 import reference_values

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _norm64(v, affine, kind, eps):
    """-> (output, error bound of an fp32 evaluation, gain / deviation of an error of the input)"""
    D = v.shape[-1]
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    dev = ((v - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    w, b = (None if t is None else t.cpu().double() for t in affine)
    w = torch.ones(D, dtype=torch.float64) if w is None else w
    n = (v - mean) / dev
    out = n * w + (0 if b is None else b)
    ulp = (D / 64 + 24) * 2.0 ** -23
    return out, ulp * (out.abs() + w.abs() * (1 + n.abs() + mean.abs() / dev)), 2 * w.abs() / dev * (1 + n.abs())


def check(got, y, r, post=None, gate=None, scale=None, pre=None, kind="layer", eps=1e-6):
    rr, h = got
    r64 = r.cpu().double()
    tol = torch.zeros_like(r64)
    if y is not None:
        z = y.cpu().double()
        ztol = torch.zeros_like(z)
        if post is not None:
            z, ztol, _ = _norm64(z, post, kind, eps)
        gs = torch.ones_like(z)
        if gate is not None:
            gt = gate.cpu().double()
            gs = gs * (gt if gt.shape == z.shape else gt.reshape(gt.shape[0], *([1] * (z.dim() - 2)), gt.shape[-1]))
        if scale is not None:
            gs = gs * scale.cpu().double()
        r64, tol = r64 + gs * z, gs.abs() * ztol + 2.0 ** -22 * (r64.abs() + (gs * z).abs())
        fi = torch.finfo(rr.dtype)
        err = (rr.cpu().double() - r64).abs()
        lim = tol + r64.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps
        assert (err <= lim).all(), float((err / lim).max())
    if pre is None:
        assert h is None
        return
    out, htol, gain = _norm64(r64, pre, kind, eps)
    htol = htol + gain * tol.amax(-1, keepdim=True)
    fi = torch.finfo(h.dtype)
    err = (h.cpu().double() - out).abs()
    lim = htol + out.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps
    assert h.shape == out.shape and (err <= lim).all(), float((err / lim).max())


def _make(shape, yt, rt, seed=0, gate=None, kind="layer"):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    y = (torch.randn(shape, generator=g) * 1.5).to(yt)
    r = (torch.randn(shape, generator=g) * 3 + 0.5 * torch.randn(D, generator=g)).to(rt)
    aff = lambda: (1 + 0.2 * torch.randn(D, generator=g), 0.1 * torch.randn(D, generator=g) if kind == "layer" else None)
    gt = None if gate is None else torch.tanh(torch.randn((shape[0], D) if gate == "row" else shape, generator=g)).to(torch.float32 if gate == "row" else yt)
    return y, r, aff(), aff(), gt, 0.1 + 0.05 * torch.randn(D, generator=g)


def _dev(t):
    return tuple(_dev(u) for u in t) if isinstance(t, tuple) else None if t is None else t.cuda()


# ------------------------------------------------------------------------------------------------------------ without a GPU
def test_refusals_before_any_launch():
    L = _lib.load()

    def call(**kw):
        a = dict(y=1 << 20, residual=1 << 21, residual_out=1 << 21, h=1 << 22, rows=4, D=32, ldy=32, ldr=32, ldro=32, ldh=32, pre=1, gate_rows=1, eps=1e-6)
        a.update(kw)
        return L.uitk_block_norm(ctypes.byref(_lib.BlockNormArgs(**a)), None)
    for kw in (dict(rows=-1), dict(D=0), dict(D=16385), dict(r_type=3), dict(y_type=3), dict(h_type=4), dict(kind=2), dict(eps=-1.0), dict(eps=float("nan")),
               dict(y=None, post=1), dict(y=None, pre=0), dict(residual=None), dict(residual_out=None), dict(h=None), dict(ldy=31), dict(ldr=31), dict(ldro=31),
               dict(ldh=31), dict(gate=1 << 23, ldg=31), dict(gate=1 << 23, ldg=32, gate_rows=0), dict(gate=1 << 23, ldg=32, gate_type=3),
               dict(h_type=3, h=(1 << 22) + 8), dict(y=(1 << 20) + 2), dict(scale=(1 << 24) + 2), dict(h=(1 << 22) + 1, h_type=1), dict(pre_w=(1 << 24) + 1)):
        assert call(**kw) == _lib.ERR_INVALID_ARG, kw
    assert call(rows=0, residual=None) == 0
    assert L.uitk_block_norm(None, None) == _lib.ERR_INVALID_ARG


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        norms.block_norm(torch.zeros(4, 32), torch.zeros(4, 32))


# ----------------------------------------------------------------------------------------------------------------------- GPU
@gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("D", [1, 2, 3, 5, 31, 64, 100, 127, 128, 129, 255, 256, 300, 512, 768, 1000, 1024, 1537, 2048, 4096, 5001, 8192, 12000, 16384])
def test_widths(D, kind):
    y, r, post, pre, gate, scale = _make((2, 3, D), torch.float32, torch.float32, seed=D, gate="row", kind=kind)
    eps = 1e-2 if D < 8 else 1e-6                                            # (tiny rows: the deviation can be as small as it likes)
    got = norms.block_norm(*_dev((y, r)), post=_dev(post), gate=_dev(gate), scale=_dev(scale), pre=_dev(pre), kind=kind, eps=eps)
    check(got, y, r, post, gate, scale, pre, kind, eps)


@gpu
@pytest.mark.parametrize("yt", DTYPES)
@pytest.mark.parametrize("rt", DTYPES)
@pytest.mark.parametrize("ht", DTYPES)
@pytest.mark.parametrize("D", [96, 770])
def test_types(yt, rt, ht, D):
    y, r, post, pre, gate, scale = _make((3, 5, D), yt, rt, seed=D, gate="token")
    got = norms.block_norm(*_dev((y, r)), post=_dev(post), gate=_dev(gate), scale=_dev(scale), pre=_dev(pre), out_dtype=ht)
    assert got[0].dtype == rt and got[1].dtype == ht
    check(got, y, r, post, gate, scale, pre)


@gpu
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "row", "token"])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 256), (4, 33, 192)])
def test_switches(post, gate, scale, pre, shape):
    y, r, po, pr, gt, sc = _make(shape, torch.bfloat16, torch.float32, seed=3, gate=gate)
    po, pr, sc = (po if post else None), (pr if pre else None), (sc if scale else None)
    got = norms.block_norm(*_dev((y, r)), post=_dev(po), gate=_dev(gt), scale=_dev(sc), pre=_dev(pr))
    check(got, y, r, po, gt, sc, pr)


@gpu
def test_first_norm_alone_gains_and_offsets_optional():
    _, r, _, pre, _, _ = _make((7, 200), torch.float32, torch.float32, seed=1)
    for p in (pre, (None, None), (pre[0], None), (None, pre[1])):
        got = norms.block_norm(None, r.cuda(), pre=_dev(p))
        check(got, None, r, pre=p)
        assert torch.equal(got[0].cpu(), r)


@gpu
@pytest.mark.parametrize("D", [32, 100, 768, 5000])
def test_four_bit_output_is_the_quantised_float_output(D):
    y, r, post, pre, gate, scale = _make((2, 70, D), torch.float32, torch.float32, seed=2, gate="row")
    kw = dict(post=_dev(post), gate=_dev(gate), scale=_dev(scale), pre=_dev(pre))
    r32, h32 = norms.block_norm(*_dev((y, r)), **kw)
    r4, h4 = norms.block_norm(*_dev((y, r)), out_dtype="mx4", **kw)
    assert torch.equal(r4, r32) and h4.shape == h32.shape
    assert torch.equal(h4.dequantize().cpu().double(), reference_values(h32))
    # the elements behind D add nothing to a product
    w = torch.randn(40, D, generator=torch.Generator().manual_seed(1)) * D ** -0.5
    wq = mx4.quantize(w.cuda())
    a, b = mx4.linear(h4, wq, out_dtype=torch.float32), mx4.linear(h32, wq, out_dtype=torch.float32)
    assert torch.allclose(a, b, rtol=0, atol=(2 * (D // 64 + 1) + 16) * 2.0 ** -22 * float((h32.abs().reshape(-1, D) @ w.cuda().abs().t()).max()) * 1.5)


@gpu
def test_inplace_and_views():
    y, r, post, pre, gate, scale = _make((2, 9, 130), torch.float16, torch.float32, seed=5, gate="row")
    want = norms.block_norm(*_dev((y, r)), post=_dev(post), gate=_dev(gate), scale=_dev(scale), pre=_dev(pre))
    wide = torch.full((2, 9, 147), 9.0, device="cuda")
    wide[..., 3:133] = r.cuda()
    view = wide[..., 3:133]
    ywide = torch.zeros((2, 9, 150), dtype=torch.float16, device="cuda")
    ywide[..., 1:131] = y.cuda()
    got = norms.block_norm(ywide[..., 1:131], view, post=_dev(post), gate=gate.cuda()[:, None], scale=_dev(scale), pre=_dev(pre), inplace=True)
    assert got[0] is view and torch.equal(view, want[0]) and torch.equal(got[1], want[1])
    assert (wide[..., :3] == 9.0).all() and (wide[..., 133:] == 9.0).all()
    same = r.cuda()
    assert torch.equal(norms.block_norm(same, same, inplace=True)[0].cpu(), r + r)


@gpu
def test_rows_do_not_mix_and_a_large_mean_survives():
    D = 512
    y, r, _, pre, _, _ = _make((40, D), torch.float32, torch.float32, seed=6)
    r[3] += 1000.0
    r[5], y[5] = 0.0, 0.0                                                    # a silent row: its deviation is sqrt(eps)
    r[7, 11] = float("nan")
    r[9, 0] = float("inf")
    got = norms.block_norm(y.cuda(), r.cuda(), pre=_dev(pre))
    h = got[1].cpu()
    assert torch.isnan(h[7]).all() and torch.isnan(h[9]).any() and not torch.isnan(h[[i for i in range(40) if i not in (7, 9)]]).any()
    keep = [i for i in range(40) if i not in (7, 9)]
    check((got[0][keep], got[1][keep]), y[keep], r[keep], pre=pre)


@gpu
def test_empty_many_rows_and_a_graph():
    assert norms.block_norm(torch.zeros(0, 64, device="cuda"), torch.zeros(0, 64, device="cuda"), pre=(None, None))[1].shape == (0, 64)
    y, r, post, pre, gate, scale = _make((257, 7, 96), torch.bfloat16, torch.bfloat16, seed=8, gate="token")
    yd, rd = _dev((y, r))
    call = lambda: norms.block_norm(yd, rd, post=_dev(post), scale=_dev(scale), pre=pd)
    pd = _dev(pre)
    post, scale = _dev(post), _dev(scale)
    want = call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for i in range(3):
        yd.copy_(torch.randn(y.shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_refusals():
    y = torch.zeros(2, 3, 64, device="cuda")
    ok = (torch.ones(64, device="cuda"), None)
    for kw, exc in ((dict(kind="batch"), ValueError), (dict(eps=-1.0), ValueError), (dict(gate=torch.zeros(3, 64, device="cuda")), ValueError),
                    (dict(scale=torch.zeros(63, device="cuda")), ValueError), (dict(post=torch.ones(64, device="cuda")), TypeError),
                    (dict(pre=(torch.ones(63, device="cuda"), None)), ValueError), (dict(pre=ok, out_dtype=torch.float64), TypeError),
                    (dict(gate=torch.zeros(2, 64)), RuntimeError)):
        with pytest.raises(exc):
            norms.block_norm(y, y.clone(), **kw)
    with pytest.raises(ValueError):
        norms.block_norm(y[:1], y)
    with pytest.raises(ValueError, match="nothing"):
        norms.block_norm(None, y)
    with pytest.raises(ValueError, match="need a block output"):
        norms.block_norm(None, y, scale=torch.zeros(64, device="cuda"), pre=ok)
    with pytest.raises(ValueError, match="in place"):
        norms.block_norm(y, torch.zeros(1, 1, 64, device="cuda").expand(2, 3, 64), inplace=True)
    flat = torch.zeros(1000, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        norms.block_norm(flat[1:385].view(2, 3, 64), flat[:384].view(2, 3, 64), inplace=True)
    with pytest.raises(RuntimeError, match="gradient"):
        norms.block_norm(y.clone().requires_grad_(), y)


@gpu
def test_offsets_past_32_bits():
    D = 4096
    rows = (1 << 31) // D + 77
    y, r = torch.zeros((rows, D), dtype=torch.bfloat16, device="cuda"), torch.zeros((rows, D), dtype=torch.bfloat16, device="cuda")
    ty, tr, _, pre, _, _ = _make((50, D), torch.bfloat16, torch.bfloat16, seed=4)
    y[-50:], r[-50:] = ty.cuda(), tr.cuda()
    got = norms.block_norm(y, r, pre=_dev(pre))
    want = norms.block_norm(ty.cuda(), tr.cuda(), pre=_dev(pre))
    assert torch.equal(got[0][-50:], want[0]) and torch.equal(got[1][-50:], want[1])


@gpu
def test_parameters_and_gates_of_other_types_and_strides():
    y, r, post, pre, gate, scale = _make((3, 4, 130), torch.float32, torch.float32, seed=9, gate="row")
    h16 = lambda t: None if t is None else t.half()
    po, pr, sc = tuple(map(h16, post)), tuple(map(h16, pre)), h16(scale)
    got = norms.block_norm(*_dev((y, r)), post=_dev(po), pre=_dev(pr), scale=torch.stack([sc, sc], 1).cuda()[:, 0], gate=gate.bfloat16().t().contiguous().cuda().t())
    check(got, y, r, tuple(t.float() for t in po), gate.bfloat16().float(), sc.float(), tuple(t.float() for t in pr))
    tok = torch.rand(3, 4, 1).expand(3, 4, 130)
    got = norms.block_norm(*_dev((y, r)), gate=tok.cuda().expand(3, 4, 130))
    check(got, y, r, gate=tok)
