"""What the operators write into a caller's tensor counts as an in-place operation on it (torch.Tensor._version)."""
import pytest
import torch

from uit_mobile_amd import mx4, norms
from uit_mobile_amd.synth import synth_pcm_i16
from test_gpu_mx4_engine import build, quiet  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_backward_pass_notices_that_what_it_saved_was_overwritten():
    x, w = torch.randn(5, 64, device="cuda"), mx4.quantize(torch.randn(48, 64, device="cuda"))
    for write in (lambda t: mx4.linear(x, w, out=t), lambda t: mx4.linear(x, w, residual=t, out=t), lambda t: norms.block_norm(x[:, :48], t, inplace=True)):
        saved, p = torch.ones(5, 48, device="cuda"), torch.ones(5, 48, device="cuda", requires_grad=True)
        loss = (saved * p).sum()
        before = saved._version
        write(saved)
        assert saved._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_calls_that_only_read_leave_the_counters_alone():
    x, w, r = torch.randn(5, 64, device="cuda"), mx4.quantize(torch.randn(64, 64, device="cuda")), torch.randn(5, 64, device="cuda")
    norms.block_norm(x, r, pre=(None, None))
    norms.block_norm(None, r, pre=(None, None), inplace=True)
    mx4.linear(x, w, residual=r)
    assert x._version == 0 and r._version == 0
    with torch.inference_mode():
        out = torch.empty(5, 64, device="cuda")
        assert mx4.linear(x, w, out=out) is out


@pytest.mark.parametrize("precision", ["mx4", "f32"])
def test_a_model_whose_parameter_was_written_is_packed_again(precision):
    m = build(precision=precision).cuda().eval()
    pcm = torch.from_numpy(synth_pcm_i16(3, 16000, seed=5)).cuda()
    bias = m.blocks[0].attn.proj.bias
    w = mx4.quantize(torch.ones(bias.numel(), 32, device="cuda"))
    with torch.no_grad():
        a = m(pcm)
        mx4.linear(torch.ones(32, device="cuda"), w, residual=bias, out=bias)
        b = m(pcm)
        m.refresh()
        assert torch.equal(b, m(pcm)) and not torch.equal(a, b)
