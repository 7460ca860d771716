"""The general engine with its dense layers on 4-bit operands (UITBase(precision='mx4'), csrc/general.hip: gen_blocks_mx4): the operators of
mx4.py and norms.py run together as the model runs them.

The engine against the same blocks composed from the public operators.  With ONE token per clip the softmax attention returns its v exactly
(one probability, 1), so the composition needs no attention of its own and both sides make the same calls; what differs is the fp32 patch
embed in front of them (another summation order: relative differences up to about 2^-20).  Such a difference moves a 4-bit code only where a
value lies within it of a rounding border; borders are at least 1/16 of a value apart, so a code moves with probability <= 2^-20 * 16 * 2 =
2^-15.  A row (one clip) passes depth * (2 dim + inner + hidden) < 2^11 roundings, so at least 15 of 16 rows are expected to have no moved code
at all; they agree to the propagated fp32 differences, bounded here by 1e-3 of the logits' scale.  A row with a moved code may be off by
what one code weighs."""
import warnings

import numpy as np
import pytest
import torch
import torch.nn as nn

from uit_mobile_amd import _lib, models, mx4, norms
from uit_mobile_amd.models.uit import UITBase, UitkSetupWarning
from uit_mobile_amd.synth import make_general_state_dict, synth_pcm_i16

gpu = pytest.mark.gpu


def build(precision="mx4", full=True, gelu=True, pooling="mean", seed=3, dim=96, heads=3, mlp_ratio=2.0, depth=3, P=16, n_mels=64, tl=102, init_values=None):
    kw = dict(outputdim=30, patch_size=P, patch_stride=P, embed_dim=dim, depth=depth, num_heads=heads, mlp_ratio=mlp_ratio, pooling=pooling, target_length=tl,
              n_mels=n_mels, attention_type="Attention" if full else "BNeckAttention", act_layer=nn.GELU if gelu else nn.ReLU, precision=precision,
              init_values=init_values)
    m = UITBase(**kw)
    sd = make_general_state_dict(embed_dim=dim, depth=depth, mlp_ratio=mlp_ratio, attention="full" if full else "bneck", patch_size=P, target_length=tl,
                                 outputdim=30, n_mels=n_mels, seed=seed)
    m.load_state_dict({k: torch.from_numpy(np.asarray(v)) for k, v in sd.items()}, strict=init_values is None)
    return m


@pytest.fixture(autouse=True)
def quiet():
    with warnings.catch_warnings():
        warnings.simplefilter("ignore", UitkSetupWarning)
        yield


def test_precision_mx4_belongs_to_the_general_engine():
    m = build()
    assert m.general and m.precision == "mx4" and m._config().precision == _lib.PREC_MX4
    with pytest.raises(NotImplementedError, match="general engine"):
        models.uit_xs(target_length=102, precision="mx4")
    with pytest.raises(NotImplementedError, match="'mx4'"):
        build(precision="fp8")


@gpu
@pytest.mark.parametrize("full,gelu,rows", [(True, True, 70), (False, False, 70), (True, False, 5), (True, True, 3000)])
def test_engine_is_the_composition_of_the_public_operators(full, gelu, rows):
    dim = 96 if full else 128
    m = build(full=full, gelu=gelu, dim=dim, heads=3 if full else 2, n_mels=16, tl=16).cuda().eval()
    x = torch.from_numpy(synth_pcm_i16(rows, 16 * 160 - 100, seed=11)).cuda()
    with torch.no_grad():
        probs, logits = m(x, return_logits=True)
        mel = m.melspec_db(x)                                                # [rows, 16, >= 16 frames]
        assert mel.shape[-1] >= 16
        bn = m.init_bn[1]
        v = (mel[..., :16] - bn.running_mean[:, None]) / torch.sqrt(bn.running_var[:, None] + 1e-5) * bn.weight[:, None] + bn.bias[:, None]
        w = m.patch_embed.proj.weight.reshape(dim, 256).double()
        r = (v.reshape(rows, 256).double() @ w.t() + m.patch_embed.proj.bias.double() + m.time_pos_embed[0, :, 0, 0].double() + m.freq_pos_embed[0, :, 0, 0].double()).float()
        inner = dim if full else dim // 4
        act = "gelu" if gelu else "relu"
        q = lambda lin: (mx4.quantize(lin.weight), lin.bias)
        _, h = norms.block_norm(None, r, pre=(m.blocks[0].norm1.weight, m.blocks[0].norm1.bias), out_dtype="mx4")
        for i, blk in enumerate(m.blocks):
            last = i + 1 == len(m.blocks)
            qkv = mx4.linear(h, q(blk.attn.qkv)[0], bias=blk.attn.qkv.bias, out_dtype=torch.float32)
            y = mx4.linear(qkv[:, 2 * inner:], q(blk.attn.proj)[0], bias=blk.attn.proj.bias)
            r, h = norms.block_norm(y, r, pre=(blk.norm2.weight, blk.norm2.bias), out_dtype="mx4", inplace=True)
            h = mx4.linear(h, q(blk.mlp.fc1)[0], bias=blk.mlp.fc1.bias, act=act, out_dtype="mx4")
            y = mx4.linear(h, q(blk.mlp.fc2)[0], bias=blk.mlp.fc2.bias)
            nxt = m.norm if last else m.blocks[i + 1].norm1
            r, h = norms.block_norm(y, r, pre=(nxt.weight, nxt.bias), out_dtype=torch.float32 if last else "mx4", inplace=True)
        hn, hl = m.outputlayer
        want = torch.nn.functional.layer_norm(h.double(), (dim,), hn.weight.double(), hn.bias.double(), hn.eps) @ hl.weight.double().t() + hl.bias.double()
    err = (logits.reshape(rows, -1).double() - want).abs().amax(-1).cpu() / float(want.abs().amax())
    assert torch.isfinite(probs).all()
    agree = float((err < 1e-3).double().mean())
    print(f"rows that agree: {agree:.4f}, median {float(err.median()):.1e}, worst {float(err.max()):.1e}")
    assert agree >= 15 / 16 if rows >= 70 else agree >= 4 / 5


@gpu
@pytest.mark.parametrize("pooling", ["mean", "token", "dm"])
def test_engine_runs_every_pooling_and_follows_the_weights(pooling):
    """Same clip, same result (in a batch of its own or not it is the same function of its codes); an edited weight is packed again."""
    m = build(pooling=pooling, full=True).cuda().eval()
    f = build(pooling=pooling, full=True, precision="f32").cuda().eval()
    x = torch.from_numpy(synth_pcm_i16(6, 16000, seed=5)).cuda()
    with torch.no_grad():
        a, ref = m(x), f(x)
        assert m.effective_precision() == "mx4" and f.effective_precision() == "f32"
        assert a.shape == ref.shape and torch.isfinite(a).all() and not torch.equal(a, ref)
        assert torch.equal(m(x), a)
        m.blocks[0].mlp.fc1.weight.mul_(0.5)
        b = m(x)
        assert not torch.equal(a, b)
        m.blocks[0].mlp.fc1.weight.mul_(2.0)
        assert torch.equal(m(x), a)


@gpu
def test_engine_layer_scale_crops_and_graph_replay():
    m = build(init_values=0.3).cuda().eval()
    T = 40000                                                                # three crops of 102 frames
    m.prepare("cuda", (5, T))
    x = torch.from_numpy(synth_pcm_i16(5, T, seed=7).astype(np.float32) / 32768.0).cuda()
    with torch.no_grad():
        want = m(x).clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m(x)
        for i in range(3):
            x.copy_(torch.from_numpy(synth_pcm_i16(5, T, seed=20 + i).astype(np.float32) / 32768.0))
            g.replay()
            got = out.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, m(x))
        assert torch.isfinite(want).all()


@gpu
def test_engine_chunks_of_its_workspace():
    """400 clips of a wide model pass the workspace in chunks; every clip's result is that of a run on fewer clips (identical calls for
    identical rows: the sums of 4-bit products round the same way unless a kernel with another order of summation takes the smaller
    batch -- allowed to move single codes, hence not compared bit for bit)."""
    m = build(dim=768, heads=12, depth=2, mlp_ratio=4.0, tl=1012).cuda().eval()
    x = torch.from_numpy(synth_pcm_i16(400, 160000, seed=2)).cuda()
    with torch.no_grad():
        a = m(x)
        b = m(x[:300])
    assert torch.isfinite(a).all()
    d = (a[:300] - b).abs().amax(-1)
    assert float((d < 1e-5).double().mean()) >= 0.5 and float(d.max()) < 0.2
