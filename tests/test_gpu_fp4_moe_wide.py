"""GPU: wide expert layers (ops/fp4.py::moe) against 64 bits, with bounds far below the outputs.

A bound that adds up the worst case of every f32 sum is as large as the output at these widths.  Here an f32 sum of K products
counts as off by at most 2^-24 (4 sqrt(K) + K / 16) of the root of its squared products: partial sums stay within a few of
those; roundings to nearest grow as sqrt(K) (four deviations), and a tensor core that cuts off instead, once per 32
products, as K / 32 steps of 2^-23.  That moves h by eh; a value of h whose e4m3 code is the same at both ends of its
interval is exact from there on, the others may be either code.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from ferrite_b200.ops import fp4  # noqa: E402
from ferrite_b200.ops import quant as Q  # noqa: E402
from test_gpu_fp4_moe import e4m3, ref_route, spread_logits  # noqa: E402

E24 = 2.0 ** -24


def random_experts(E, D, I, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    q = lambda std, *s: fp4.quantize(torch.randn(*s, generator=g, device="cuda") * std)
    return q(D ** -0.5, E, 2, I, D), q(I ** -0.5, E, D, I)


def values(t, e):
    return fp4.reference_dequantize(fp4.Fp4Tensor(t.codes[e], t.scales[e], t.fmt, t.shape[1:], t.tensor_scale))


def grow(K):
    return E24 * (4 * math.sqrt(K) + K / 16)


def reference(x, logits, w13, w2, topk, bias, score, norm, scale, limit):
    """(y, element bound, row bound): rows add the independent changes of h in quadrature, twice."""
    idx, w = ref_route(logits.cpu(), None if bias is None else bias.cpu(), topk, score, norm, scale)
    D, I, T = x.shape[1], w2.shape[2], x.shape[0]
    xq = Q.fp8_act_roundtrip(torch.nn.functional.pad(x.float().cpu(), (0, -D % 32))).double()[:, :D].cuda()
    y, tol, sq, own = (torch.zeros(T, D, dtype=torch.float64, device="cuda") for _ in range(4))
    b = lambda v: v.view(-1, 32)
    for e in idx.unique().tolist():
        W13, W2 = values(w13, e), values(w2, e)
        for t, k in (idx == e).nonzero().tolist():
            wt = float(w[t, k])
            (g, u), (eg, eu) = (W13 @ xq[t]), grow(D) * ((W13 * xq[t]) ** 2).sum(-1).sqrt()
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
            s = g * torch.sigmoid(g)
            h = s * u * wt
            eh = abs(wt) * (1.1 * eg * (u.abs() + eu) + s.abs() * eu) + 32 * E24 * h.abs() + 1e-12
            amax, ea = b(h.abs()).amax(-1, keepdim=True), b(eh).amax(-1, keepdim=True)
            q = e4m3(b(h).cpu(), amax.cpu()).view(-1).cuda()
            alts = [e4m3(b(h + sg * eh).cpu(), (amax + sa * ea).cpu()).view(-1).cuda() for sg in (-1, 1) for sa in (-1, 1)]
            dq = torch.stack([(a - q).abs() for a in alts]).amax(0)
            y[t] += W2 @ q
            tol[t] += W2.abs() @ dq
            sq[t] += W2 ** 2 @ dq ** 2
            own[t] += W2 ** 2 @ (q.abs() + dq) ** 2
    down = grow(topk * I + 256) * own.sqrt()
    return y, tol + down, 2 * sq.sum(1).sqrt() + down.norm(dim=1)


CASES = [  # T, E, topk, D, I, score, norm, bias, dtype of x
    (2, 16, 6, 5120, 2304, "sqrtsoftplus", True, True, torch.bfloat16),   # the production width
    (8, 24, 6, 5120, 576, "sqrtsoftplus", True, True, torch.float32),     # its quarter
    (4, 6, 2, 5120, 288, "sqrtsoftplus", True, True, torch.bfloat16),
    (20, 4, 2, 7168, 128, "sigmoid", True, False, torch.bfloat16),
    (2, 6, 2, 5120, 64, "sigmoid", False, True, torch.float32),           # few tiles: clusters of eight
    (24, 16, 2, 2048, 512, "softmax", True, True, torch.bfloat16),
    (12, 9, 3, 3200, 96, "sqrtsoftplus", True, True, torch.float16),      # an odd number of 128-column blocks
    (8, 24, 6, 8192, 32, "sigmoid", True, True, torch.bfloat16),          # the widest rows
    (32, 5, 2, 8192, 64, "softmax", True, True, torch.float32),
    (32, 40, 6, 5120, 320, "sqrtsoftplus", True, True, torch.bfloat16),
    (17, 12, 4, 5000, 416, "sigmoid", True, True, torch.bfloat16),        # nothing is a multiple of 128
]


@pytest.mark.parametrize("T,E,topk,D,I,score,norm,with_bias,dtype", CASES)
def test_wide_layers(T, E, topk, D, I, score, norm, with_bias, dtype):
    g = torch.Generator().manual_seed(T * 1000 + I)
    w13, w2 = random_experts(E, D, I, I)
    x = (torch.randn(T, D, generator=g) * torch.logspace(-0.5, 0.5, T).unsqueeze(1)).to(dtype).cuda()
    logits = spread_logits(T, E, I).cuda()
    bias = (torch.randperm(E, generator=g).float() * 0.37 / E).cuda() if with_bias else None
    kw = dict(bias=bias, score=score, norm=norm, scale=1.5, limit=4.0)
    y, tol, row = reference(x, logits, w13, w2, topk, **kw)
    size = y.norm(dim=1)
    # The bounds say something.  One value of h between two codes moves its row by up to 2^-3 |h| of its norm, counted twice: where
    # a row has a few hundred values the largest is up to half of that norm, which makes 1/8.
    assert (row <= 0.15 * size).all() and (row / size).median() <= 0.04 and (tol.norm(dim=1) <= 0.5 * size).all()
    got = fp4.moe(x, logits, w13, w2, topk, out_dtype=torch.float32, **kw).double()
    fp4.check()
    assert ((got - y).norm(dim=1) <= row).all(), float(((got - y).norm(dim=1) / size).max())
    assert ((got - y).abs() <= tol).all(), float(((got - y).abs() - tol).max())
    low = fp4.moe(x, logits, w13, w2, topk, out_dtype=torch.bfloat16, **kw)
    assert torch.equal(low, fp4.moe(x, logits, w13, w2, topk, out_dtype=torch.float32, **kw).bfloat16())


def test_the_bounds_see_a_misplaced_scale_block():
    """What the layer would give with two neighbouring scale blocks of one expert's matrix exchanged lies outside the bounds
    (the mistake is planted in the statement)."""
    T, E, topk, D, I = 2, 4, 2, 5120, 320
    w13, w2 = random_experts(E, D, I, 1)
    x = torch.randn(T, D, generator=torch.Generator().manual_seed(1)).cuda()
    logits = spread_logits(T, E, 1).cuda()
    kw = dict(bias=None, score="sigmoid", norm=True, scale=1.0, limit=4.0)
    got = fp4.moe(x, logits, w13, w2, topk, out_dtype=torch.float32, **kw).double()
    e = int(logits[0].argmax())
    for which in (0, 1):
        parts = [fp4.Fp4Tensor(t.codes, t.scales.clone(), t.fmt, t.shape) for t in (w13, w2)]
        s = parts[which].scales[e].flatten(0, -3)      # [row tiles, chunks, 512]
        rows = s.view(-1, s.shape[-2], 32, 4, 4)
        rows[:, 1, :, :, 0], rows[:, 1, :, :, 1] = rows[:, 1, :, :, 1] + 1, rows[:, 1, :, :, 0] + 1
        y, tol, row = reference(x, logits, *parts, topk, **kw)
        assert ((got - y).norm(dim=1)[0] > row[0]) and not ((got - y)[0].abs() <= tol[0]).all()
    y, tol, row = reference(x, logits, w13, w2, topk, **kw)
    assert ((got - y).norm(dim=1) <= row).all()
