"""The general engine between its two stages: what a front-end call left behind is not used once its buffer has been replaced."""
import pytest
import torch

from uit_mobile_amd.synth import synth_pcm_i16
from test_gpu_mx4_engine import build, quiet  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("precision", ["f32", "mx4"])
def test_a_larger_reservation_between_the_stages_is_noticed(precision):
    m = build(precision=precision).cuda().eval()
    x = torch.from_numpy(synth_pcm_i16(4, 16000, seed=5)).cuda()
    with torch.no_grad():
        want = m(x)
        state = m.frontend(x)
        m.reserve(2, 16000)                                                  # nothing grows: the state stays good
        assert torch.equal(m.encode(state), want)
        state = m.frontend(x)
        m.reserve(64, 16000)                                                 # the frames are gone
        with pytest.raises(ValueError, match="no front-end output"):
            m.encode(state)
        assert torch.equal(m(x), want) and torch.equal(m.encode(m.frontend(x)), want)


@pytest.mark.parametrize("precision", ["f32", "mx4"])
def test_a_growth_that_a_capture_refuses_leaves_the_state_good(precision):
    m = build(precision=precision).cuda().eval()
    x, more = (torch.from_numpy(synth_pcm_i16(n, 16000, seed=5)).cuda() for n in (4, 64))
    with torch.no_grad():
        want = m(x)
        state = m.frontend(x)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            with pytest.raises(RuntimeError, match="workspace has to grow"):
                with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
                    m(more)
        torch.cuda.synchronize()
        assert torch.equal(m.encode(state), want)
