"""The GELU of mx4.linear by itself: with a zero product its input is the bias.

Tolerance 2^-21 max(1, |y|): the fitted polynomial 7e-8; then, relative to y, the logit (three roundings, times at most 0.28: |logit| (1 - Phi) is
no larger) 5e-8, the exponential 2^-24, the sum 2^-24, the reciprocal 2^-23 and the last product 2^-24: 7e-8 + 3.5e-7 |y| < 2^-21 max(1, |y|)."""
import pytest
import torch

from uit_mobile_amd import mx4

gpu = pytest.mark.gpu


def inputs():
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.linspace(-14, 14, 150001), 3 * torch.randn(100000, generator=g), torch.exp2(torch.empty(6000).uniform_(-126, 20, generator=g)),
                   -torch.exp2(torch.empty(6000).uniform_(-126, 20, generator=g))])
    return torch.cat([x, torch.tensor([0.0, -0.0, 5.5, -5.5, 3e38, -3e38, float("inf"), float("nan")])])


@gpu
@pytest.mark.parametrize("rows", [1, 65])                                    # the rows kernels, the tile kernels
def test_gelu_is_within_its_bound(rows):
    x = inputs()
    n = x.numel()
    w = mx4.quantize(torch.zeros(n, 32, device="cuda"))
    got = mx4.linear(torch.zeros(rows, 32, device="cuda"), w, bias=x.cuda(), act="gelu").cpu()
    assert torch.equal(got.nan_to_num(7.0), got[:1].nan_to_num(7.0).expand(rows, n))
    y = got[0].double()
    want = x.double() * torch.special.ndtr(x.double())
    finite = torch.isfinite(x)
    err = (y - want).abs()[finite] / want.abs()[finite].clamp(min=1.0)
    print(f"largest error {float(err.max()):.2e} max(1, |y|) at x = {float(x[finite][err.argmax()]):.4f}")
    assert float(err.max()) < 2.0 ** -21
    assert y[-1].isnan() and y[-2] == float("inf") and float(y[-4].float()) == float(torch.tensor(3e38)) and y[-3] == 0.0
    assert not got[0, -8:-6].any()                                            # (+0: a bias of -0 is added to a product of +0)
