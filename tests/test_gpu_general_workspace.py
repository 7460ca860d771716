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


@pytest.mark.parametrize("precision", ["f32", "mx4"])
@pytest.mark.parametrize("T", [16000, 40000])                                # one crop, three crops
def test_a_graph_keeps_its_buffers_when_a_larger_batch_grows_them(precision, T):
    m = build(precision=precision).cuda().eval()
    m.prepare("cuda", (4, T), dtype=torch.int16)
    x, more = (torch.from_numpy(synth_pcm_i16(n, T, seed=5)).cuda() for n in (4, 200))
    with torch.no_grad():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m(x)
        for i in range(3):
            big = m(more[:100 * (i + 1) if i < 2 else 200])                  # grows, grows again, stays
            keep = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(4)]     # what a freed buffer would be given to
            x.copy_(torch.from_numpy(synth_pcm_i16(4, T, seed=30 + i)))
            g.replay()
            got = out.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, m(x)) and torch.isfinite(big).all() and len(keep) == 4
