"""Views whose memory is not their values: the imaginary part of a conjugate is a real tensor with a negative bit (torch.Tensor.is_neg), stored with
the other sign.  Exact comparisons: the operators have to see the same numbers."""
import pytest
import torch

from uit_mobile_amd import mx4, norms
from uit_mobile_amd.mx4 import as_rows

gpu = pytest.mark.gpu
SHAPES = [(1, 1), (5, 1), (2, 3, 1), (1, 8), (5, 40), (2, 3, 40)]


def imag_of_conjugate(shape, device="cpu"):
    t = torch.randn(shape, dtype=torch.cfloat, generator=torch.Generator().manual_seed(sum(shape))).to(device).conj().imag
    assert t.is_neg()
    return t


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_handed_to_a_kernel_hold_the_values(shape):
    for t in (imag_of_conjugate(shape), torch.randn(shape), torch.randn(shape[:-1] + (shape[-1] + 3,))[..., :shape[-1]], torch.randn(shape[:1] + (1,) * (len(shape) - 1)).expand(shape)):
        K = shape[-1]
        v, ld = as_rows(t, K)
        rows = t.numel() // K
        raw = torch.as_strided(v, (rows, K), (ld, 1))
        assert not v.is_neg() and (rows == 1 or ld >= K) and torch.equal(raw, t.reshape(rows, K))


@gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_operators_see_the_values(shape):
    t, K = imag_of_conjugate(shape, "cuda"), shape[-1]
    plain = torch.empty(shape, device="cuda").copy_(t)
    assert not plain.is_neg() and torch.equal(plain, t)
    assert torch.equal(mx4.quantize(t).dequantize(), mx4.quantize(plain).dequantize())
    w = mx4.quantize(torch.ones(4, K, device="cuda"))
    assert torch.equal(mx4.linear(t, w), mx4.linear(plain, w))
    one = mx4.quantize(torch.ones(1, K, device="cuda"))
    res = imag_of_conjugate(shape[:-1] + (1,), "cuda")
    bias = imag_of_conjugate((1,), "cuda")
    assert torch.equal(mx4.linear(plain, one, bias=bias, residual=res), mx4.linear(plain, one, bias=bias.resolve_neg(), residual=res.resolve_neg()))
    vec = imag_of_conjugate((K,), "cuda")
    got = norms.block_norm(t, t, pre=(vec, vec), scale=vec, kind="rms", gate=t)
    want = norms.block_norm(plain, plain, pre=(vec.resolve_neg(), vec.resolve_neg()), scale=vec.resolve_neg(), kind="rms", gate=plain)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if K == 1 and plain.numel() == 1:
        with pytest.raises(ValueError, match="contiguous"):
            mx4.linear(plain, one, out=res)
