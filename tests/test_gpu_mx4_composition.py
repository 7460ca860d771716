"""The general engine in precision 'mx4' on clips of several tokens, against the same network composed from the public operators (mx4.py, norms.py)
and the textbook attention in 64 bits: softmax over tokens, its scale, the cls token, the three poolings, crops, and LayerScale gains folded into
the rows of a weight before it is rounded to 4 bits.

What may differ.  Everything between two 4-bit roundings is fp32 in the engine and 32 or 64 bits here: relative differences up to about 2^-20 of
a row's scale.  Such a difference moves a 4-bit code where a value lies within it of a rounding border; borders are at least 1/16 of the block's
largest value apart, so a code moves with probability <= 2^-20 * 16 * 2 = 2^-15.  A clip passes tokens * depth * (2 dim + inner + hidden) * crops
roundings: at most 5 * 2 * 320 and 4 * 2 * 320 * 3 < 7700 here, so at most 7700 * 2^-15 < 1/4 of the clips are expected to have a moved code;
asserted is a third, three standard deviations of 200 clips above that.  The others agree to the propagated fp32 differences, bounded
by 1e-3 of the logits' scale (1e-3 of a probability: its slope in the logit is at most 1/4 and the logits here reach 4 and more)."""
import warnings

import pytest
import torch

from uit_mobile_amd import mx4, norms
from uit_mobile_amd.models.uit import UitkSetupWarning
from uit_mobile_amd.synth import synth_pcm_i16
from test_gpu_mx4_engine import build

pytestmark = pytest.mark.gpu

CLIPS, TL, N_MELS, P = 200, 32, 32, 16                                       # 2 x 2 patches of a crop


def crops_of(v, crops, tl):
    """[B, mels, frames] -> [B * crops, mels, tl]: consecutive crops, the last one the clip's last frames"""
    if crops == 1:
        return v
    parts = [v[..., i * tl:(i + 1) * tl] for i in range(crops - 1)] + [v[..., -tl:]]
    return torch.stack(parts, 1).flatten(0, 1)


def compose(m, x):
    """-> (probabilities [B, C], logits [B * crops, C] or None for pooling 'dm')"""
    dim, heads, crops = m.embed_dim, m.num_heads, m.num_crops(x.shape[1])
    bn = m.init_bn[1]
    mel = m.melspec_db(x).double()
    v = (mel - bn.running_mean[:, None]) / torch.sqrt(bn.running_var[:, None].double() + 1e-5) * bn.weight[:, None] + bn.bias[:, None]
    v = crops_of(v, crops, TL)
    nt = v.shape[-1] // P
    rows, gf = v.shape[0], N_MELS // P
    patches = v[..., :nt * P].reshape(rows, gf, P, nt, P).permute(0, 1, 3, 2, 4).reshape(rows, gf, nt, P * P)
    w = m.patch_embed.proj.weight.reshape(dim, P * P).double()
    r = patches @ w.t() + m.patch_embed.proj.bias + m.time_pos_embed[0, :, 0, :nt].t().double() + m.freq_pos_embed[0, :, :, 0].t().double()[:, None]
    r = r.reshape(rows, gf * nt, dim)
    if m.pooling == "token":
        r = torch.cat([(m.cls_token + m.token_pos_embed).double().expand(rows, 1, dim), r], 1)
    r = r.float()
    T = r.shape[1]
    inner = dim if m.attention_full else dim // 4
    hd = inner // heads
    act = "gelu" if m.act_gelu else "relu"

    def folded(lin, ls):
        """weight (4-bit) and bias behind a LayerScale gain"""
        if not m.init_values:
            return mx4.quantize(lin.weight), lin.bias
        g = ls.gamma.double()
        return mx4.quantize((lin.weight.double() * g[:, None]).float()), (lin.bias.double() * g).float()
    _, h = norms.block_norm(None, r, pre=(m.blocks[0].norm1.weight, m.blocks[0].norm1.bias), out_dtype="mx4")
    for i, blk in enumerate(m.blocks):
        last = i + 1 == len(m.blocks)
        qkv = mx4.linear(h, mx4.quantize(blk.attn.qkv.weight), bias=blk.attn.qkv.bias, out_dtype=torch.float32)
        q, k, u = qkv.double().view(rows, T, 3, heads, hd).permute(2, 0, 3, 1, 4)                      # [rows, heads, T, hd] each
        s = (q[..., :, None, :] * k[..., None, :, :]).sum(-1) * (dim // heads) ** -0.5
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = ((e / e.sum(-1, keepdim=True))[..., None] * u[..., None, :, :]).sum(-2)
        o = o.permute(0, 2, 1, 3).reshape(rows, T, inner).float()
        wq, b = folded(blk.attn.proj, blk.ls1)
        r, h = norms.block_norm(mx4.linear(o, wq, bias=b), r, pre=(blk.norm2.weight, blk.norm2.bias), out_dtype="mx4")
        h = mx4.linear(h, mx4.quantize(blk.mlp.fc1.weight), bias=blk.mlp.fc1.bias, act=act, out_dtype="mx4")
        wq, b = folded(blk.mlp.fc2, blk.ls2)
        nxt = m.norm if last else m.blocks[i + 1].norm1
        r, h = norms.block_norm(mx4.linear(h, wq, bias=b), r, pre=(nxt.weight, nxt.bias), out_dtype=torch.float32 if last else "mx4")
    h = h.double()
    if m.pooling == "token":
        z = h[:, 0]
    elif m.pooling == "mean":
        z = h.mean(1)
    else:
        z = h.view(rows, gf, nt, dim).mean(1)                                # a group per time patch
    hn, hl = m.outputlayer
    z = torch.nn.functional.layer_norm(z, (dim,), hn.weight.double(), hn.bias.double(), hn.eps)
    logits = z @ hl.weight.double().t() + hl.bias.double()
    probs = torch.sigmoid(logits)
    if m.pooling == "dm":
        probs, logits = probs.mean(1), None
    return probs.view(-1, crops, probs.shape[-1]).mean(1), logits


CASES = {
    "mean": dict(),
    "token": dict(pooling="token"),
    "dm": dict(pooling="dm"),
    "layer_scale": dict(init_values=0.5),
    "bneck_relu_token_layer_scale": dict(pooling="token", full=False, gelu=False, dim=128, mlp_ratio=1.0, init_values=0.5),
    "crops": dict(crops=3),
    "crops_dm_layer_scale": dict(pooling="dm", init_values=0.5, crops=3),
}


@pytest.mark.parametrize("name", list(CASES))
def test_engine_is_the_network_composed_of_the_operators(name):
    kw = dict(CASES[name])
    crops = kw.pop("crops", 1)
    m = build(**{**dict(dim=64, heads=2, depth=2, mlp_ratio=2.0, n_mels=N_MELS, tl=TL), **kw}).cuda().eval()
    g = torch.Generator().manual_seed(8)
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore", UitkSetupWarning)
        if m.init_values:                                                    # gains of 1/4 .. 2 and both signs, another one per channel
            for blk in m.blocks:
                for ls in (blk.ls1, blk.ls2):
                    ls.gamma.copy_(torch.exp2(3 * torch.rand(m.embed_dim, generator=g) - 2) * torch.where(torch.rand(m.embed_dim, generator=g) < 0.2, -1.0, 1.0))
        T = (TL * crops - (0 if crops == 1 else 16)) * 160 - 100             # (the last crop overlaps the one before)
        x = torch.from_numpy(synth_pcm_i16(CLIPS, T, seed=11)).cuda()
        assert m.num_crops(T) == crops
        want, want_logits = compose(m, x)
        if want_logits is None:
            got, logits = m(x), None
        else:
            got, logits = m(x, return_logits=True)
    assert got.shape == want.shape and torch.isfinite(got).all()
    err = (got.double() - want).abs().amax(-1)
    ok = err < 1e-3
    if logits is not None:
        e = (logits.reshape(want_logits.shape).double() - want_logits).abs().amax(-1) / want_logits.abs().amax()
        ok &= (e.view(CLIPS, crops) < 1e-3).all(-1)
        assert float(want_logits.abs().amax()) >= 4.0
    agree = float(ok.double().mean())
    print(f"{name}: clips that agree {agree:.3f}, median {float(err.median()):.1e}, worst {float(err.max()):.1e}")
    assert agree >= 2 / 3
