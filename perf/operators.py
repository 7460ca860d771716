"""What is timed of the microscaled 4-bit operators and of the fused block norms, on one MI355X.

Three operators, reached through `uit_mobile_amd.mx4` and `uit_mobile_amd.norms`:

* quantize  a matrix [rows, K] -> 4-bit floating point in blocks of 32 consecutive elements of a row that share a power-of-two scale
            (OCP MXFP4: elements e2m1, scale e8m0), and back to the values those codes stand for;
* linear    out = residual + act(Q(x) . W^T + bias), Q(x) the 4-bit rounding of the activations (or activations that are 4-bit already),
            W [N, K] weights that a program quantises once and keeps;
* norm      the seam between two blocks of a transformer: r' = r + gate * scale * post_norm(y), h = pre_norm(r').

With `own` false every operator is computed in its plain form: elementary torch operations in 32 bits, rounded once at the end.

The MXFP4 rounding of a block v[0..31] (all arithmetic of it is exact in 32 bits): with e = floor(log2(max |v|)) the scale is 2^X,
X = max(e - 2, -127); an element is v / 2^X rounded to the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ties to the even code, values
beyond 6 to 6.  The last block of a row is short where K is no multiple of 32.
"""
import math

import torch

own = False

BLOCK = 32
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "mx4": 0.5 + 1.0 / BLOCK}

_LARGEST_QUANTIZE = 32768 * 4096           # elements
_LARGEST_LINEAR = 8192 ** 3                # multiply-adds
_LARGEST_NORM = 8 * 4096 * 4096            # elements


def listed():
    return [
        # one embedding vector on its way into a 4-bit layer: the latency of the smallest call
        dict(name="quantize_one_token", op="quantize", rows=1, K=768, dtype="f32", pad=0),
        # attention outputs of a ragged batch, a width that is no multiple of a block
        dict(name="quantize_ragged", op="quantize", rows=1021, K=1000, dtype="f16", pad=24),
        # the activations of a large batch (or a weight matrix at load time): bandwidth
        dict(name="quantize_largest", op="quantize", rows=32768, K=4096, dtype="bf16", pad=0),
        # the query / key / value layer of the default UITBase (768 wide) for a single token
        dict(name="linear_one_token", op="linear", M=1, N=2304, K=768, x="bf16", out="bf16", bias=True, act=None, residual=False, pad=0),
        # a dozen rows against a large weight matrix: reading the weights is all there is
        dict(name="linear_few_rows", op="linear", M=13, N=8192, K=8192, x="bf16", out="bf16", bias=True, act="relu", residual=False, pad=0),
        # the attention's output layer of the default UITBase, one 10 s clip (4 x 63 patches), added onto its fp32 residual stream
        dict(name="linear_one_clip", op="linear", M=252, N=768, K=768, x="f32", out="f32", bias=True, act=None, residual=True, pad=0),
        # nothing is a multiple of anything: the 537 classes, rows inside a wider buffer
        dict(name="linear_ragged", op="linear", M=1003, N=537, K=1000, x="f16", out="f16", bias=True, act="gelu", residual=False, pad=8),
        # the query / key / value layer of the default UITBase, 64 clips at once, activations 4-bit already (they left the norm that way)
        dict(name="linear_batch", op="linear", M=16128, N=2304, K=768, x="mx4", out="bf16", bias=True, act=None, residual=False, pad=0),
        # a large square layer: the matrix pipes
        dict(name="linear_largest", op="linear", M=8192, N=8192, K=8192, x="bf16", out="bf16", bias=True, act="gelu", residual=False, pad=0),
        # the seam between two blocks for one token, everything switched on
        dict(name="norm_one_token", op="norm", B=1, T=1, D=768, y="f32", r="f32", out="f32", kind="layer", post=True, gate="row", scale=True, pre=True, pad=0),
        # the default UITBase, 64 clips: layer-scaled attention output added to the fp32 stream, the MLP's LayerNorm behind it
        dict(name="norm_batch", op="norm", B=64, T=252, D=768, y="f32", r="f32", out="f32", kind="layer", post=False, gate=None, scale=True, pre=True, pad=0),
        # a wide 16-bit stream, root-mean-square norms before and after, a gate per sequence
        dict(name="norm_largest", op="norm", B=8, T=4096, D=4096, y="bf16", r="bf16", out="bf16", kind="rms", post=True, gate="row", scale=True, pre=True, pad=0),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v))


def _width(rng, lo, hi):
    """A width: any whole number, or (as often) a multiple of 32, as model widths mostly are."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < 0.5 else max(32, v // 32 * 32)


def draw(rng):
    """One more case of the same ranges: rows 1 .. 65536, widths 16 .. 8192, every type and every switch."""
    op = rng.choice(["quantize", "linear", "linear", "norm"])
    pad = rng.choice([0, 0, 0, 8, 17])
    if op == "quantize":
        K = _width(rng, 16, 8192)
        rows = _log_int(rng, 1, min(65536, _LARGEST_QUANTIZE // K))
        return dict(op=op, rows=rows, K=K, dtype=rng.choice(["f32", "f16", "bf16"]), pad=pad)
    if op == "linear":
        N, K = _width(rng, 16, 8192), _width(rng, 16, 8192)
        M = _log_int(rng, 1, min(32768, _LARGEST_LINEAR // (N * K)))
        x = rng.choice(["f32", "f16", "bf16", "mx4"])
        return dict(op=op, M=M, N=N, K=K, x=x, out=rng.choice(["f32", "f16", "bf16"]), bias=rng.random() < 0.7,
                    act=rng.choice([None, "relu", "gelu"]), residual=rng.random() < 0.3, pad=0 if x == "mx4" else pad)
    D = _width(rng, 16, 8192)
    tokens = _log_int(rng, 1, min(65536, _LARGEST_NORM // D))
    B = _log_int(rng, 1, min(64, tokens))
    y = rng.choice(["f32", "f16", "bf16"])
    return dict(op=op, B=B, T=max(1, tokens // B), D=D, y=y, r=rng.choice(["f32", y]), out=rng.choice(["f32", "f16", "bf16"]),
                kind=rng.choice(["layer", "rms"]), post=rng.random() < 0.5, gate=rng.choice([None, "row", "token"]), scale=rng.random() < 0.6,
                pre=rng.random() < 0.8, pad=pad)


# ------------------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, K, dtype, pad):
    """What a norm or an activation function hands to a layer: unit-sized values, a few channels much larger than the others, a few
    silent rows.  `pad` more columns in memory: the rows of a slice of a wider buffer."""
    full = torch.empty((rows, K + pad), dtype=_TYPES[dtype], device="cuda")
    channel = torch.exp(0.5 * _normal(g, 1, K))
    channel = torch.where(torch.rand((1, K), generator=g, device="cuda") < 0.01, channel * 20.0, channel)
    quiet = torch.where(torch.rand((rows, 1), generator=g, device="cuda") < 0.02, 0.0, 1.0)
    for r0 in range(0, rows, 8192):
        r1 = min(rows, r0 + 8192)
        full[r0:r1, :K] = (_normal(g, r1 - r0, K) * channel * quiet[r0:r1]).to(_TYPES[dtype])
    if pad:
        full[:, K:] = 7.0
    return full[:, :K]


def _inputs(case, seed):
    g = _gen(seed)
    if case["op"] == "quantize":
        return dict(x=_activations(g, case["rows"], case["K"], case["dtype"], case["pad"]))
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        d = dict(x=_activations(g, M, K, "bf16" if case["x"] == "mx4" else case["x"], case["pad"]),
                 w=_normal(g, N, K) * (K ** -0.5), bias=None, residual=None)
        if case["bias"]:
            d["bias"] = 0.1 * _normal(g, N)
        if case["residual"]:
            d["residual"] = _normal(g, M, N).to(_TYPES[case["out"]])
        return d
    B, T, D = case["B"], case["T"], case["D"]
    d = dict(y=_activations(g, B * T, D, case["y"], case["pad"]).view(B, T, D) if case["pad"] == 0 else
             _activations(g, B * T, D, case["y"], case["pad"]).unflatten(0, (B, T)),
             r=(_normal(g, B, T, D) * 3.0 + 0.5 * _normal(g, 1, 1, D)).to(_TYPES[case["r"]]), post=None, gate=None, scale=None, pre=None)
    affine = (lambda: (1.0 + 0.2 * _normal(g, D), 0.1 * _normal(g, D) if case["kind"] == "layer" else None))
    if case["post"]:
        d["post"] = affine()
    if case["gate"] == "row":
        d["gate"] = torch.tanh(_normal(g, B, D))
    elif case["gate"] == "token":
        d["gate"] = torch.sigmoid(_normal(g, B, T, D)).to(_TYPES[case["y"]])
    if case["scale"]:
        d["scale"] = 0.1 + 0.05 * _normal(g, D)
    if case["pre"]:
        d["pre"] = affine()
    return d


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["op"] == "linear":
        # the weights are 4-bit from the moment the program loads them (the plain form keeps the values they stand for)
        if own:
            from uit_mobile_amd import mx4
            state["w"] = mx4.quantize(state["w"])
            if case["x"] == "mx4":
                state["x"] = mx4.quantize(state["x"])
        else:
            state["w"] = _round_mx4(state["w"])
            if case["x"] == "mx4":
                state["x"] = _round_mx4(state["x"])
    return state


# ------------------------------------------------------------------------------------------------------------------- plain forms
def _round_mx4(x):
    """The values (float32) of the MXFP4 codes of x [rows, K], by comparison with the midpoints between neighbouring codes."""
    rows, K = x.shape
    v = x.to(torch.float32)
    short = -K % BLOCK
    if short:
        v = torch.cat([v, v.new_zeros((rows, short))], 1)
    v = v.view(rows, -1, BLOCK)
    a = v.abs()
    _, e = torch.frexp(a.amax(-1, keepdim=True))                    # amax = m 2^e, m in [0.5, 1): floor(log2 amax) = e - 1
    X = (e - 3).clamp_(min=-127)
    y = a * _power_of_two(-X)
    q = 0.5 * (y > 0.25) + 0.5 * (y >= 0.75) + 0.5 * (y > 1.25) + 0.5 * (y >= 1.75) + 1.0 * (y > 2.5) + 1.0 * (y >= 3.5) + 2.0 * (y > 5.0)
    q = torch.copysign(0.5 * q, v) * _power_of_two(X + 1)
    return q.view(rows, -1)[:, :K]


def _power_of_two(n):
    """2^n, n = -126 .. 127, from its bits"""
    return ((n + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_linear(s):
    x = s["x"] if s["case"]["x"] == "mx4" else _round_mx4(s["x"])
    y = x @ s["w"].t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["case"]["act"] == "relu":
        y = torch.clamp(y, min=0.0)
    elif s["case"]["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if s["residual"] is not None:
        y = s["residual"].to(torch.float32) + y
    return y.to(_TYPES[s["case"]["out"]])


def _plain_norm(v, affine, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    v = v * affine[0]
    return v if affine[1] is None else v + affine[1]


EPS = 1e-6


def _plain_block_norm(s):
    c = s["case"]
    z = s["y"].to(torch.float32)
    if s["post"] is not None:
        z = _plain_norm(z, s["post"], c["kind"], EPS)
    if s["gate"] is not None:
        z = z * (s["gate"].to(torch.float32) if c["gate"] == "token" else s["gate"][:, None, :])
    if s["scale"] is not None:
        z = z * s["scale"]
    r = s["r"].to(torch.float32) + z
    h = None if s["pre"] is None else _plain_norm(r, s["pre"], c["kind"], EPS).to(_TYPES[c["out"]])
    return (r.to(_TYPES[c["r"]]),) if h is None else (r.to(_TYPES[c["r"]]), h)


def run(state):
    c = state["case"]
    if not own:
        if c["op"] == "quantize":
            return _round_mx4(state["x"]).to(_TYPES["f32" if c["dtype"] == "f16" else c["dtype"]])
        return _plain_linear(state) if c["op"] == "linear" else _plain_block_norm(state)
    if c["op"] == "quantize":
        from uit_mobile_amd import mx4
        # (a block scale of f16 data can be too small for f16 itself: those values come back in 32 bits)
        return mx4.quantize(state["x"]).dequantize(_TYPES["f32" if c["dtype"] == "f16" else c["dtype"]])
    if c["op"] == "linear":
        from uit_mobile_amd import mx4
        return mx4.linear(state["x"], state["w"], bias=state["bias"], act=c["act"], residual=state["residual"], out_dtype=_TYPES[c["out"]])
    from uit_mobile_amd import norms
    r, h = norms.block_norm(state["y"], state["r"], post=state["post"], gate=state["gate"], scale=state["scale"], pre=state["pre"],
                            kind=c["kind"], eps=EPS, out_dtype=_TYPES[c["out"]])
    return (r,) if h is None else (r, h)


# ------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Each input once, each output once.  quantize: the input, the packed codes and scales, and the values; flops: the products of a
    linear layer, about 2 / 16 operations an element of a quantisation / a norm."""
    if case["op"] == "quantize":
        n = case["rows"] * case["K"]
        out = _SIZE["f32" if case["dtype"] == "f16" else case["dtype"]]
        return {"bytes": n * (_SIZE[case["dtype"]] + _SIZE["mx4"] + out), "flops": 2.0 * n}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        b = M * K * _SIZE[case["x"]] + N * K * _SIZE["mx4"] + M * N * _SIZE[case["out"]] * (2 if case["residual"] else 1) + (4 * N if case["bias"] else 0)
        return {"bytes": b, "flops": 2.0 * M * N * K}
    B, T, D = case["B"], case["T"], case["D"]
    n = B * T * D
    b = n * (_SIZE[case["y"]] + 2 * _SIZE[case["r"]] + (_SIZE[case["out"]] if case["pre"] else 0))
    b += {None: 0, "row": 4 * B * D, "token": n * _SIZE[case["y"]]}[case["gate"]]
    b += 4 * D * ((2 if case["post"] else 0) + (2 if case["pre"] else 0) + (1 if case["scale"] else 0))
    return {"bytes": b, "flops": 16.0 * n}


# ------------------------------------------------------------------------------------------------------- the definition, 64 bits
def _exact_mx4(x):
    """MXFP4 by its grid: the codes of one binade are evenly spaced (0.5 up to 2, 1 up to 4, 2 up to 6), so the nearest code is a
    rounding to a multiple of the spacing, ties to the even multiple."""
    rows, K = x.shape
    out = torch.empty((rows, K), dtype=torch.float64, device=x.device)
    for k0 in range(0, K, BLOCK * 32):
        v = x[:, k0:k0 + BLOCK * 32].to(torch.float64)
        n = v.shape[1]
        v = torch.nn.functional.pad(v, (0, -n % BLOCK)).reshape(rows, -1, BLOCK)
        top = v.abs().max(-1, keepdim=True).values
        expo = (top.view(torch.int64) >> 52) - 1023                               # the exponent field: floor(log2), -1023 for zero
        unit = (((expo - 2).clamp(min=-127) + 1023) << 52).view(torch.float64)
        y = v / unit
        spacing = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
        y = (torch.round(y / spacing) * spacing).clamp(-6.0, 6.0) * unit
        out[:, k0:k0 + n] = y.reshape(rows, -1)[:, :n]
    return out


def _exact_linear(c, d):
    w = _exact_mx4(d["w"])
    outs = []
    step = max(1, min(c["M"], (1 << 27) // max(c["N"], c["K"])))
    for m0 in range(0, c["M"], step):
        y = torch.matmul(_exact_mx4(d["x"][m0:m0 + step]), w.T)
        if d["bias"] is not None:
            y += d["bias"].double()
        if c["act"] == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif c["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        if d["residual"] is not None:
            y = y + d["residual"][m0:m0 + step].double()
        outs.append(y)
    return torch.cat(outs)


def _exact_norm(v, affine, kind):
    if kind == "layer":
        var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
        v = (v - mean) / torch.sqrt(var + EPS)
    else:
        v = v / torch.sqrt(v.square().sum(-1, keepdim=True) / v.shape[-1] + EPS)
    v = affine[0].double() * v
    return v if affine[1] is None else v + affine[1].double()


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "quantize":
        return _exact_mx4(d["x"])
    if case["op"] == "linear":
        return _exact_linear(case, d)
    rs, hs = [], []
    for b in range(case["B"]):
        z = d["y"][b].double()
        if d["post"] is not None:
            z = _exact_norm(z, d["post"], case["kind"])
        if d["gate"] is not None:
            z = z * d["gate"][b].double()
        if d["scale"] is not None:
            z = d["scale"].double() * z
        r = d["r"][b].double() + z
        rs.append(r)
        if d["pre"] is not None:
            hs.append(_exact_norm(r, d["pre"], case["kind"]))
    return (torch.stack(rs), torch.stack(hs)) if hs else (torch.stack(rs),)
