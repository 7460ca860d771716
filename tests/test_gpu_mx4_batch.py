"""The general engine in precision 'mx4': a clip's result does not depend on the calls, shards or chunks it shares -- bit for bit, as in every
other precision.  A product's rows are independent, so this asks that the order in which a product adds does not depend on how many rows it
has: a last bit moves 4-bit codes further down, and those move the result by what 4 bits cost.

(Products of two 4-bit values are multiples of 1/4 up to 36: where the block scales of a row are alike, a sum of a few thousand of them fits fp32
exactly, and any order gives the same bits.  So the models here have channels of very different sizes, as trained ones do.)"""
import pytest
import torch

from uit_mobile_amd.synth import synth_pcm_i16
from test_gpu_mx4_engine import build, quiet  # noqa: F401  (the fixture that silences the set-up warning)

pytestmark = pytest.mark.gpu

GEOMETRIES = {
    "one_token": (dict(n_mels=16, tl=16, dim=384, heads=6, mlp_ratio=4.0), 2000, 16 * 160 - 100),                  # a row a clip
    "wide_hidden": (dict(n_mels=16, tl=16, dim=1024, heads=8, depth=1, mlp_ratio=4.0), 16384, 16 * 160 - 100),     # the largest tiles
    "default_width": (dict(dim=768, heads=12, depth=2, mlp_ratio=4.0, tl=1012), 40, 160000),                       # 248 tokens a clip
    "bneck_relu_cls_crops": (dict(dim=256, heads=2, full=False, gelu=False, pooling="token", init_values=0.3), 80, 40000),   # three crops
    "dm": (dict(dim=192, pooling="dm"), 400, 16000),
}


def uneven(m):
    """Channels of very different sizes: every 32 of the norms' outputs, of the attention's values and of the MLP's hidden layer times a power of two."""
    g = torch.Generator().manual_seed(4)

    def powers(n):
        return 2.0 ** -torch.randint(0, 25, (-(-n // 32),), generator=g).float().repeat_interleave(32)[:n]
    with torch.no_grad():
        for b in m.blocks:
            for norm in (b.norm1, b.norm2):
                p = powers(norm.weight.numel())
                norm.weight.mul_(p)
                norm.bias.mul_(p)
            inner = b.attn.proj.weight.shape[1]
            for lin, lo, n in ((b.attn.qkv, 2 * inner, inner), (b.mlp.fc1, 0, b.mlp.fc1.weight.shape[0])):
                p = powers(n)
                lin.weight[lo:lo + n].mul_(p[:, None])
                lin.bias[lo:lo + n].mul_(p)
    return m


@pytest.mark.parametrize("name", list(GEOMETRIES))
def test_a_clip_does_not_see_the_batch_it_is_in(name):
    """The top_db floor is the batch's, as in the reference: the sub-batches get the whole batch's maximum, as a data-parallel run gives it."""
    kw, B, T = GEOMETRIES[name]
    m = uneven(build(**kw)).cuda().eval()
    x = torch.from_numpy(synth_pcm_i16(min(B, 512), T, seed=9)).cuda()
    x = x.repeat(-(-B // x.shape[0]), 1)[:B]
    top = []
    with torch.no_grad():
        want = m(x, amax_sync=lambda slots: top.append(slots.max().clone()))
        assert torch.isfinite(want).all()
        for lo, hi in ((0, 1), (5, 6), (0, 3), (7, 16), (0, B // 2), (B // 2, B), (1, B)):
            got = m(x[lo:hi], amax_sync=lambda slots: slots.copy_(top[0].expand(64)))
            assert torch.equal(got, want[lo:hi]), (name, lo, hi, float((got - want[lo:hi]).abs().max()))


@pytest.mark.parametrize("T,crops,copies", [(160000, 1, 44), (320000, 2, 22)])
def test_every_clip_of_every_chunk_is_that_clip_alone(T, crops, copies):
    """More rows (a clip's crop each) than the engine's 3 GiB workspace takes at once: 704 of the default width in two chunks, the second
    one short, their border inside a copy of the clips and inside a clip's crops.  Sixteen clips many times over: every copy has the bits of
    the sixteen by themselves."""
    m = uneven(build(dim=768, heads=12, depth=2, mlp_ratio=4.0, tl=1012)).cuda().eval()
    tokens = 4 * ((1012 if crops > 1 else m.num_frames(T)) // 16)
    floats = 16 * 16 + 2 * 768 + 3 * 768 + 768                             # fp32 work buffers of a token
    per_chunk = (3 << 30) // (tokens * floats * 4)
    rows = 16 * crops * copies
    assert m.num_crops(T) == crops and per_chunk < rows < 2 * per_chunk and per_chunk % (16 * crops) and (crops == 1 or per_chunk % crops)
    few = torch.from_numpy(synth_pcm_i16(16, T, seed=2)).cuda()
    with torch.no_grad():
        want, want_logits = m(few, return_logits=True)
        got, got_logits = m(few.repeat(copies, 1), return_logits=True)
    assert torch.isfinite(want).all()
    assert torch.equal(got.view(copies, 16, -1), want.expand(copies, 16, -1))
    assert torch.equal(got_logits.reshape(copies, 16, -1), want_logits.reshape(1, 16, -1).expand(copies, 16, -1))
