"""Cases of the block-scaled 4-bit operators (``ferrite_b200.ops.fp4``) and their plain forms.

Three operators, as a program that serves a model with 4-bit weights calls them:

* ``roundtrip``: a matrix is quantised (``fp4.quantize``) and expanded again (``fp4.dequantize``).  The codes and scales
  are 4- and 8-bit, so what comes back is the values they stand for.
* ``linear``: ``fp4.linear`` quantises the rows of ``x`` and multiplies them with 4-bit weights.
* ``moe``: ``fp4.moe``, a whole layer of 4-bit experts for a few tokens: routing from the router's logits, gate and up
  products, SwiGLU, down product and the weighted sum over the chosen experts.

Formats.  A value is an e2m1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and sign; two codes a byte, the even column in the low
nibble) times the scale of its block of consecutive columns.  ``mxfp4``: blocks of 32, scale a power of two (ue8m0
byte), ``2^ceil(log2(amax / 6))``.  ``nvfp4``: blocks of 16, scale an e4m3 number, ``amax / 6`` rounded, and one f32
scale for the whole tensor by which the values are divided first (rounded to f32).  Rows are padded with zero codes to whole groups of
128 columns, and so are their scales; the scale bytes of 128 rows and 4 blocks form a chunk of 512 bytes, byte ``16 i + 4 g + s`` for row
``32 g + i`` and block ``s``.
"""
import torch

own = False

_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of odd rows on their way into a 4-bit cache: the smallest call, where the launch counts
        {"name": "roundtrip 16x1000 nv f16", "op": "roundtrip", "fmt": "nvfp4", "rows": 16, "cols": 1000, "src": "f16", "dst": "f16"},
        # one expert's down projection converted from f32 at load time
        {"name": "roundtrip 5120x2304 mx f32", "op": "roundtrip", "fmt": "mxfp4", "rows": 5120, "cols": 2304, "src": "f32", "dst": "bf16"},
        # a layer's fused input projection converted at load time, with a scale for the whole tensor
        {"name": "roundtrip 24896x4096 nv bf16", "op": "roundtrip", "fmt": "nvfp4", "rows": 24896, "cols": 4096, "src": "bf16", "dst": "bf16"},
        # decode of one sequence: the attention output projection
        {"name": "linear 1x8192x5120 mx", "op": "linear", "fmt": "mxfp4", "rows": 1, "cols": 8192, "outs": 5120, "src": "bf16", "dst": "bf16"},
        # a batched decode step: the fused input projection, whose width is no multiple of a tile
        {"name": "linear 16x4096x24896 nv", "op": "linear", "fmt": "nvfp4", "rows": 16, "cols": 4096, "outs": 24896, "src": "bf16", "dst": "bf16"},
        # sizes that fit nothing: rows, columns and outputs all end inside a tile
        {"name": "linear 333x1000x1111 nv f16", "op": "linear", "fmt": "nvfp4", "rows": 333, "cols": 1000, "outs": 1111, "src": "f16", "dst": "f16"},
        # a prefill chunk through a gate | up projection, f32 activations as this framework's layers hand them over
        {"name": "linear 1024x5120x4608 mx f32", "op": "linear", "fmt": "mxfp4", "rows": 1024, "cols": 5120, "outs": 4608, "src": "f32", "dst": "bf16"},
        # a long prefill through the widest projection: the largest product
        {"name": "linear 8192x4096x24896 nv", "op": "linear", "fmt": "nvfp4", "rows": 8192, "cols": 4096, "outs": 24896, "src": "bf16", "dst": "bf16"},
        # decode of one sequence through the routed experts of a layer
        {"name": "moe 1 token", "op": "moe", "tokens": 1, "experts": 384, "topk": 6, "dim": 5120, "inter": 2304, "score": "sqrtsoftplus", "src": "bf16", "dst": "bf16"},
        # a speculative draft block through the draft layers' smaller expert set
        {"name": "moe 5 tokens draft", "op": "moe", "tokens": 5, "experts": 128, "topk": 3, "dim": 5120, "inter": 2304, "score": "sqrtsoftplus", "src": "bf16", "dst": "bf16"},
        # a batched tick on one of four tensor-parallel ranks: each holds a quarter of every expert's columns
        {"name": "moe 8 tokens shard", "op": "moe", "tokens": 8, "experts": 384, "topk": 6, "dim": 5120, "inter": 576, "score": "sqrtsoftplus", "src": "f32", "dst": "bf16"},
        # a batched tick of 32 sequences with sigmoid routing
        {"name": "moe 32 tokens", "op": "moe", "tokens": 32, "experts": 384, "topk": 6, "dim": 5120, "inter": 2304, "score": "sigmoid", "src": "bf16", "dst": "bf16"},
    ]


def _size(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread evenly over its logarithm."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    return max(step, v // step * step)


def draw(rng):
    op = rng.choice(("roundtrip", "linear", "linear", "moe"))
    fmt = rng.choice(("mxfp4", "nvfp4"))
    if op == "roundtrip":
        return {"op": op, "fmt": fmt, "rows": _size(rng, 1, 24896), "cols": _size(rng, 16, 4096),
                "src": rng.choice(("bf16", "f16", "f32")), "dst": rng.choice(("bf16", "f16"))}
    if op == "linear":
        src = rng.choice(("bf16", "f16", "f32"))
        return {"op": op, "fmt": fmt, "rows": _size(rng, 1, 8192), "cols": _size(rng, 64, 4096), "outs": _size(rng, 32, 24896),
                "src": src, "dst": "f16" if src == "f16" else "bf16"}
    experts = rng.choice((128, 256, 288, 384))
    return {"op": op, "tokens": _size(rng, 1, 32), "experts": experts, "topk": rng.choice((1, 2, 3, 4, 6)),
            "dim": _size(rng, 512, 5120, 128), "inter": _size(rng, 256, 2304, 32),
            "score": rng.choice(("sqrtsoftplus", "sigmoid", "softmax")), "src": rng.choice(("bf16", "f16", "f32")), "dst": "bf16"}


def _groups(cols):
    return (cols + 127) // 128


def work(case):
    """Each input read once, each output written once; of the experts, those that the tokens choose (at most)."""
    size = {"bf16": 2, "f16": 2, "f32": 4}
    a, b = size[case["src"]], size[case["dst"]]
    if case["op"] == "moe":
        t, d, i = case["tokens"], case["dim"], case["inter"]
        pairs = t * case["topk"]
        # experts hit by `pairs` picks, as many as independent picks hit on average
        hit = case["experts"] * (1 - (1 - case["topk"] / case["experts"]) ** t)
        return {"bytes": hit * 3 * d * i * 17 / 32 + t * d * (a + b) + t * case["experts"] * 4, "flops": 2 * pairs * 3 * d * i}
    n, k = case["rows"], case["cols"]
    per = 0.5 + 1 / _BLOCK[case["fmt"]]
    if case["op"] == "roundtrip":
        return {"bytes": n * k * (a + 2 * per + b), "flops": 4 * n * k}
    m = case["outs"]
    return {"bytes": n * k * a + m * k * per + n * m * b, "flops": 2 * n * k * m}


# ---- inputs --------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _to_chunks(s):
    """Scale bytes [..., rows, blocks] -> [..., ceil(rows / 128), ceil(blocks / 4), 512]."""
    rows, blocks = s.shape[-2:]
    s = torch.nn.functional.pad(s, (0, -blocks % 4, 0, -rows % 128))
    lead = s.shape[:-2]
    s = s.reshape(*lead, s.shape[-2] // 128, 4, 32, s.shape[-1] // 4, 4)
    n = len(lead)
    return s.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).reshape(*lead, s.shape[n], s.shape[n + 3], 512).contiguous()


def _random_weights(shape, fmt, g, std):
    """4-bit weights as a checkpoint holds them: codes and scale chunks, of about N(0, std) values."""
    *lead, rows, cols = shape
    codes = torch.randint(0, 256, (*lead, rows, 64 * _groups(cols)), dtype=torch.uint8, device="cuda", generator=g)
    real = torch.arange(64 * _groups(cols), device="cuda") * 2
    codes = torch.where(real + 1 < cols, codes, torch.where(real < cols, codes & 15, codes & 0))
    blocks = 128 * _groups(cols) // _BLOCK[fmt]
    if fmt == "mxfp4":  # the codes' own spread is about 2.9
        s = (torch.randint(0, 2, (*lead, rows, blocks), device="cuda", generator=g, dtype=torch.uint8)
             + (126 + round(torch.log2(torch.tensor(std / 2.9)).item())))
        return codes, _to_chunks(s), None
    s = torch.randint(32, 120, (*lead, rows, blocks), device="cuda", generator=g, dtype=torch.uint8)
    return codes, _to_chunks(s), std / 2.9 / 64


def prepare(case, seed):
    g = _gen(seed)
    src = _TYPES[case["src"]]
    if case["op"] == "moe":
        t, e, d, i = case["tokens"], case["experts"], case["dim"], case["inter"]
        s = {"x": torch.randn(t, d, device="cuda", generator=g).to(src),
             "logits": torch.randn(t, e, device="cuda", generator=g) * 2,
             "bias": torch.randn(e, device="cuda", generator=g) * 0.05}
        s["w13"] = _random_weights((e, 2, i, d), "mxfp4", g, d ** -0.5)
        s["w2"] = _random_weights((e, d, i), "mxfp4", g, i ** -0.5)
        s["case"] = case
        return s
    n, k = case["rows"], case["cols"]
    x = torch.randn(n, k, device="cuda", generator=g)
    # rows of unlike size, as activations after a gate and rows of a weight matrix are
    x = x * torch.exp(torch.randn(n, 1, device="cuda", generator=g) * 0.5)
    if case["op"] == "roundtrip":
        x = (x * 0.02).to(src)
        ts = float(x.float().abs().max() / (6 * 448)) if case["fmt"] == "nvfp4" else None  # an f32 number
        return {"x": x, "ts": ts, "case": case}
    return {"x": x.to(src), "w": _random_weights((case["outs"], k), case["fmt"], g, k ** -0.5), "case": case}


# ---- plain forms ---------------------------------------------------------------------------------
def _lut(dtype=torch.float32):
    v = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device="cuda")
    return torch.stack([v.repeat(16), v.repeat_interleave(16)], 1)  # by byte: (even column, odd column)


def _scale_values(byte, fmt):
    if fmt == "nvfp4":
        return byte.view(torch.float8_e4m3fn).float()
    return (byte.int() << 23).view(torch.float32)


def _from_chunks(c, rows, blocks):
    lead = c.shape[:-3]
    n = len(lead)
    c = c.reshape(*lead, c.shape[n], c.shape[n + 1], 32, 4, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    return c.reshape(*lead, c.shape[n] * 128, -1)[..., :rows, :blocks]


def _values(codes, chunks, fmt, rows, cols):
    """f32 values [..., rows, cols] of codes and scale chunks."""
    b = _BLOCK[fmt]
    v = _lut()[codes.int()].flatten(-2)
    s = _scale_values(_from_chunks(chunks, rows, v.shape[-1] // b), fmt)
    return (v.unflatten(-1, (-1, b)) * s.unsqueeze(-1)).flatten(-2)[..., :cols]


def _pow2_ceil(x):
    m, e = torch.frexp(x)
    return ((torch.where(m == 0.5, e - 1, e) + 127) << 23).view(torch.float32)  # as bits: a power function may be an ulp off


def _blocks(x, b):
    k = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -k % b)).unflatten(-1, (-1, b))


def _e2m1(a):
    """Nearest of the eight magnitudes, ties to the even code."""
    return (0.5 * ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5).float() + (a >= 3.5)
            + 2.0 * (a > 5.0))


def _fp4_values(x, fmt, ts=None):
    """The values that quantised x stands for (before the tensor's own scale is put back)."""
    u = x.float() if ts is None else (x.double() / torch.full((), ts, dtype=torch.float64, device="cuda")).float()
    v = _blocks(u, _BLOCK[fmt])
    amax = v.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        s = _pow2_ceil(amax.clamp_min(6 * 2.0 ** -126) * (torch.ones_like(amax) / 6))
    else:
        # next to the border of two scales: the quotient itself, not a product with the reciprocal
        s = (amax.clamp_min(6 * 2.0 ** -9).double() / torch.full((), 6.0, device="cuda")).clamp_max(448).float().to(torch.float8_e4m3fn).float()
    q = v / s
    return (torch.copysign(_e2m1(q.abs()), q) * s).flatten(-2)[..., : x.shape[-1]]


def _fp8_values(x):
    """e4m3 with a power-of-two scale for each 32 values, as activations meet 4-bit experts."""
    v = _blocks(x.float(), 32)
    s = _pow2_ceil(v.abs().amax(-1, keepdim=True).clamp_min(1e-4) * (torch.ones(1, device="cuda") / 448))
    return ((v / s).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s).flatten(-2)[..., : x.shape[-1]]


def _route(logits, bias, topk, score):
    """Chosen experts [tokens, topk] and their weights; the bias counts for the choice alone."""
    z = logits.double()  # next to the border of the choice 32 bits would not decide
    p = {"sqrtsoftplus": lambda: (z.clamp_min(0) + torch.log1p(torch.exp(-z.abs()))).sqrt(), "sigmoid": lambda: 1 / (1 + torch.exp(-z)),
         "softmax": lambda: torch.exp(z - z.amax(-1, keepdim=True)) / torch.exp(z - z.amax(-1, keepdim=True)).sum(-1, keepdim=True)}[score]()
    idx = torch.sort(p + bias.double(), dim=-1, descending=True, stable=True).indices[:, :topk]
    w = p.gather(1, idx)
    return idx, (w / w.sum(-1, keepdim=True) * 1.5).float()


def _moe(s, case):
    d, i = case["dim"], case["inter"]
    idx, w = _route(s["logits"], s["bias"], case["topk"], case["score"])
    e = idx.flatten()
    x = _fp8_values(s["x"]).repeat_interleave(case["topk"], 0)
    w13 = _values(s["w13"][0][e], s["w13"][1][e], "mxfp4", i, d)
    gate, up = torch.einsum("pgik,pk->gpi", w13, x)
    del w13
    gate, up = gate.clamp(max=10.0), up.clamp(-10.0, 10.0)
    h = _fp8_values(gate / (1 + torch.exp(-gate)) * up * w.flatten()[:, None])
    y = torch.einsum("pdi,pi->pd", _values(s["w2"][0][e], s["w2"][1][e], "mxfp4", d, i), h)
    return y.unflatten(0, (-1, case["topk"])).sum(1).to(_TYPES[case["dst"]])


def run(state):
    case = state["case"]
    dst = _TYPES[case["dst"]]
    if own:
        from ferrite_b200.ops import fp4
        if case["op"] == "roundtrip":
            return fp4.dequantize(fp4.quantize(state["x"], case["fmt"], tensor_scale=state["ts"]), dst)
        if case["op"] == "linear":
            codes, chunks, ts = state["w"]
            w = fp4.Fp4Tensor(codes, chunks, case["fmt"], (case["outs"], case["cols"]), ts)
            return fp4.linear(state["x"], w, out_dtype=dst)
        e, d, i = case["experts"], case["dim"], case["inter"]
        w13 = fp4.Fp4Tensor(*state["w13"][:2], "mxfp4", (e, 2, i, d))
        w2 = fp4.Fp4Tensor(*state["w2"][:2], "mxfp4", (e, d, i))
        return fp4.moe(state["x"], state["logits"], w13, w2, case["topk"], bias=state["bias"], score=case["score"],
                       scale=1.5, limit=10.0, out_dtype=dst)
    if case["op"] == "roundtrip":
        ts = state["ts"]
        v = _fp4_values(state["x"], case["fmt"], ts)
        return (v if ts is None else v * ts).to(dst)
    if case["op"] == "linear":
        codes, chunks, ts = state["w"]
        w = _values(codes, chunks, case["fmt"], case["outs"], case["cols"])
        y = _fp4_values(state["x"], case["fmt"]) @ w.t()
        return (y if ts is None else y * ts).to(dst)
    return _moe(state, case)


# ---- the definition in 64 bits -------------------------------------------------------------------
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _two_to(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_weights(codes, chunks, fmt, rows, cols):
    grid = torch.tensor(_GRID, dtype=torch.float64, device="cuda")
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :cols]
    v = grid[(nib & 7).long()] * (1 - 2 * (nib >> 3).double())
    r, c = torch.arange(rows, device="cuda")[:, None], torch.arange(cols, device="cuda")[None, :] // _BLOCK[fmt]
    byte = chunks[r // 128, c // 4, r % 32 * 16 + r % 128 // 32 * 4 + c % 4]
    if fmt == "mxfp4":
        return v * _two_to(byte.long() - 127)
    m, e = (byte & 7).double(), (byte >> 3 & 15).double()
    return v * torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * _two_to(e - 7))


def _round_float(v, mant, emin, top):
    """v rounded to a binary number of `mant` fraction bits (ties to even), subnormal below 2^emin, at most `top`."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** (emin - 4)))).clamp_min(emin)
    step = _two_to(e - mant)
    return (torch.round(v / step) * step).clamp(-top, top)


def _exact_quant(x, fmt, ts=None):
    b = {"e4m3": 32, **_BLOCK}[fmt]
    # what is left of a value by the tensor's scale is an f32 number: the blocks' scales and codes are defined on that
    u = x.double() if ts is None else (x.double() / torch.full((), ts, dtype=torch.float64, device="cuda")).float().double()
    k = u.shape[-1]
    v = torch.cat([u, u.new_zeros(*u.shape[:-1], -k % b)], -1).reshape(*u.shape[:-1], -1, b)
    top = v.abs().max(-1, keepdim=True).values
    if fmt == "nvfp4":
        s = _round_float(top.clamp_min(6 * 2.0 ** -9) / torch.full_like(top, 6.0), 3, -6, 448.0)
    else:
        most, floor = (6.0, 6 * 2.0 ** -126) if fmt == "mxfp4" else (448.0, 1e-4)
        s = _two_to(torch.ceil(torch.log2(top.clamp_min(floor) / most)))
    q = _round_float(v / s, 3, -6, 448.0) if fmt == "e4m3" else _round_float(v / s, 1, 0, 6.0)
    return (q * s).reshape(*u.shape[:-1], -1)[..., :k]


def _exact_moe(s, case):
    z, topk, d, i = s["logits"].double(), case["topk"], case["dim"], case["inter"]
    if case["score"] == "softmax":
        p = torch.softmax(z, -1)
    elif case["score"] == "sigmoid":
        p = torch.sigmoid(z)
    else:
        p = torch.logaddexp(z, torch.zeros_like(z)).sqrt()
    pick = (-(p + s["bias"].double())).argsort(dim=-1, stable=True)[:, :topk]
    x = _exact_quant(s["x"], "e4m3")
    y = x.new_zeros(x.shape)
    for t, row in enumerate(pick.tolist()):
        total = p[t, pick[t]].sum()
        for e in row:
            gate = (_exact_weights(s["w13"][0][e, 0], s["w13"][1][e, 0], "mxfp4", i, d) @ x[t]).clamp(max=10.0)
            up = (_exact_weights(s["w13"][0][e, 1], s["w13"][1][e, 1], "mxfp4", i, d) @ x[t]).clamp(-10.0, 10.0)
            h = _exact_quant(gate * torch.sigmoid(gate) * up * (1.5 * p[t, e] / total), "e4m3")
            y[t] += _exact_weights(s["w2"][0][e], s["w2"][1][e], "mxfp4", d, i) @ h
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "moe":
        return _exact_moe(s, case)
    if case["op"] == "roundtrip":
        return _exact_quant(s["x"], case["fmt"], s["ts"]) * (1.0 if s["ts"] is None else s["ts"])
    codes, chunks, ts = s["w"]
    w = _exact_weights(codes, chunks, case["fmt"], case["outs"], case["cols"])
    return _exact_quant(s["x"], case["fmt"]) @ w.t() * (1.0 if ts is None else ts)
