"""GPU: the expert layer for a few tokens (ops/fp4.py::moe) against a plain statement in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from ferrite_b200.ops import fp4  # noqa: E402
from ferrite_b200.ops import quant as Q  # noqa: E402

E24 = 2.0 ** -24


def experts(E, D, I, seed=0):
    g = torch.Generator().manual_seed(seed)
    w13 = fp4.quantize((torch.randn(E, 2, I, D, generator=g) * D ** -0.5).cuda())
    w2 = fp4.quantize((torch.randn(E, D, I, generator=g) * I ** -0.5).cuda())
    return w13, w2


def spread_logits(T, E, seed=0):
    """Logits of every token in a random order of values well apart: no choice hangs on a rounding."""
    g = torch.Generator().manual_seed(seed + 1)
    grid = torch.linspace(-3.0, 3.0, E)
    return torch.stack([grid[torch.randperm(E, generator=g)] for _ in range(T)])


def ref_route(logits, bias, topk, score, norm, scale):
    z = logits.double()
    p = {"sqrtsoftplus": lambda: torch.nn.functional.softplus(z).sqrt(), "sigmoid": lambda: torch.sigmoid(z),
         "softmax": lambda: torch.softmax(z, -1)}[score]()
    key = z if bias is None else p + bias.double()
    key = torch.where(torch.isnan(key), torch.full_like(key, -math.inf), key)
    idx = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :topk]
    w = p.gather(1, idx)
    if norm:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return idx, w * scale


def e4m3(v, amax):
    s = Q.pow2_ceil((amax.clamp_min(1e-4) * Q._INV448).float()).double()
    return Q.e4m3_round((v / s).float()).double() * s


def ref_moe(x, logits, w13, w2, topk, bias=None, score="sqrtsoftplus", norm=True, scale=1.0, limit=0.0):
    """(y, tol): the layer in 64 bits, and how far an evaluation in f32 may be from it.  An f32 sum of K products is off by
    at most (K + 2) half steps of the absolute sum; that (through SwiGLU, whose slope is below 1.1) moves h by at most eh,
    and where h +- eh rounds to different e4m3 values the down product may see either."""
    x, logits = x.cpu(), logits.cpu()
    bias = None if bias is None else bias.cpu()
    idx, w = ref_route(logits, bias, topk, score, norm, scale)
    xq = Q.fp8_act_roundtrip(torch.nn.functional.pad(x.float(), (0, -x.shape[1] % 32))).double()[:, :x.shape[1]]
    W13, W2 = fp4.reference_dequantize(w13).cpu(), fp4.reference_dequantize(w2).cpu()
    I, D = W13.shape[2], W13.shape[3]
    y, tol = torch.zeros(x.shape[0], D, dtype=torch.float64), torch.zeros(x.shape[0], D, dtype=torch.float64)
    lim = limit if limit else math.inf
    for t in range(x.shape[0]):
        mag = torch.zeros(D, dtype=torch.float64)
        for k in range(topk):
            e = int(idx[t, k])
            g, u = W13[e, 0] @ xq[t], W13[e, 1] @ xq[t]
            eg, eu = ((D + 2) * E24 * (W13[e, j].abs() @ xq[t].abs()) for j in (0, 1))
            g, u = g.clamp(max=lim), u.clamp(-lim, lim)
            s = g * torch.sigmoid(g)
            h = s * u * w[t, k]
            eh = w[t, k].abs() * (1.1 * eg * (u.abs() + eu) + s.abs() * eu) + 32 * E24 * h.abs() + 1e-12
            b = lambda v: v.view(-1, 32)
            amax, ea = b(h.abs()).amax(-1, keepdim=True), b(eh).amax(-1, keepdim=True)
            q = e4m3(b(h), amax).view(-1)
            alts = [e4m3(b(h + sg * eh), amax + sa * ea).view(-1) for sg in (-1, 1) for sa in (-1, 1)]
            dq = torch.stack([(a - q).abs() for a in alts]).amax(0)
            y[t] += W2[e] @ q
            tol[t] += W2[e].abs() @ dq
            mag += W2[e].abs() @ (q.abs() + dq)
        tol[t] += (topk * I + 8) * E24 * mag
    return y, tol


def check_close(got, y, tol, dtype):
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    err = (got.cpu().double() - y).abs()
    lim = tol * (1 + eps) + eps * y.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert (err <= lim).all(), (float(err.max()), float((err - lim).max()))


CASES = [  # T, E, topk, D, I, score, norm, bias, dtype
    (1, 8, 2, 256, 64, "sqrtsoftplus", True, True, torch.bfloat16),
    (1, 384, 6, 512, 128, "sqrtsoftplus", True, False, torch.float32),
    (1, 1, 1, 128, 32, "softmax", False, False, torch.float32),
    (3, 16, 4, 1000, 96, "sigmoid", True, True, torch.float16),
    (5, 12, 3, 1280, 576, "sqrtsoftplus", False, True, torch.float32),
    (16, 20, 3, 384, 160, "softmax", True, True, torch.bfloat16),
    (17, 40, 6, 640, 256, "sigmoid", False, False, torch.float32),
    (32, 64, 8, 130, 32, "softmax", True, False, torch.float16),
    (32, 33, 32, 96, 64, "sqrtsoftplus", True, True, torch.bfloat16),
    (2, 512, 6, 256, 32, "sigmoid", True, True, torch.float32),
    (4, 6, 2, 5120, 288, "sqrtsoftplus", True, True, torch.bfloat16),
    (20, 4, 2, 7168, 128, "sigmoid", True, False, torch.bfloat16),
    (2, 6, 2, 5120, 64, "sigmoid", False, True, torch.float32),        # few tiles: clusters of eight
    (24, 16, 2, 2048, 512, "softmax", True, True, torch.bfloat16),     # clusters of two
    (12, 9, 3, 3200, 96, "sqrtsoftplus", True, True, torch.float16),   # an odd number of 128-column blocks
    (32, 96, 6, 1024, 256, "sqrtsoftplus", True, False, torch.bfloat16),
    (8, 24, 6, 8192, 32, "sigmoid", True, True, torch.bfloat16),       # the widest rows
    (32, 5, 2, 8192, 64, "softmax", True, True, torch.float32),
]


@pytest.mark.parametrize("T,E,topk,D,I,score,norm,with_bias,dtype", CASES)
def test_moe(T, E, topk, D, I, score, norm, with_bias, dtype):
    g = torch.Generator().manual_seed(T * 100 + E)
    w13, w2 = experts(E, D, I, T)
    x = (torch.randn(T, D, generator=g) * torch.logspace(-1, 1, T).unsqueeze(1)).to(dtype).cuda()
    logits = spread_logits(T, E, E).cuda()
    bias = (torch.randperm(E, generator=g).float() * 0.37 / E).cuda() if with_bias else None
    kw = dict(bias=bias, score=score, norm=norm, scale=1.5, limit=2.0)
    got = fp4.moe(x, logits, w13, w2, topk, **kw)
    fp4.check()
    assert got.dtype == dtype
    y, tol = ref_moe(x, logits, w13, w2, topk, **kw)
    check_close(got, y, tol, dtype)
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        check_close(fp4.moe(x, logits, w13, w2, topk, out_dtype=out_dtype, **kw), y, tol, out_dtype)


def test_route_edges():
    """Ties go to the lower index, masked experts (the type's lowest value, -inf) and NaN come last, one token's NaN
    stays in its row, a token of zeros gives zeros."""
    E, D, I, topk = 40, 256, 64, 3
    w13, w2 = experts(E, D, I, 5)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(8, D, generator=g)
    logits = spread_logits(8, E, 3)
    logits[0] = 0.0                                          # all equal
    logits[1] = -math.inf
    logits[1, [30, 7, 19]] = torch.tensor([0.0, -5.0, 2.0])  # exactly topk left
    logits[2] = torch.finfo(torch.float32).min
    logits[2, [1, 39]] = 1.0                                 # fewer than topk left: the lowest masked index joins
    logits[3, 5:] = math.nan
    logits[4, 9] = math.inf
    x[5], x[6, 200] = 0.0, math.nan
    for score in ("sigmoid", "sqrtsoftplus"):
        got = fp4.moe(x.cuda(), logits.cuda(), w13, w2, topk, score=score, norm=False, limit=1.0).cpu()
        rows = [0, 1, 2, 3, 5, 7] + ([4] if score == "sigmoid" else [])
        y, tol = ref_moe(x[rows], logits[rows], w13, w2, topk, score=score, norm=False, limit=1.0)
        check_close(got[rows], y, tol, torch.float32)
        assert (got[5] == 0).all() and torch.isnan(got[6]).all()
        assert torch.isfinite(got[rows]).all()


def test_every_token_takes_the_same_expert_and_none_do():
    E, D, I = 9, 512, 96
    w13, w2 = experts(E, D, I, 6)
    x = torch.randn(32, D, generator=torch.Generator().manual_seed(2)).cuda()
    same = torch.zeros(32, E, device="cuda")
    same[:, 4] = 3.0
    apart = torch.zeros(32, E, device="cuda")
    apart[torch.arange(32), torch.arange(32) % E] = 3.0
    for logits in (same, apart):
        got = fp4.moe(x, logits, w13, w2, 1, score="sigmoid", norm=True)
        check_close(got, *ref_moe(x, logits, w13, w2, 1, score="sigmoid"), torch.float32)


def test_strided_tensors_accumulate_and_rows_left_alone():
    T, E, D, I, topk = 6, 16, 384, 64, 4
    w13, w2 = experts(E, D, I, 7)
    g = torch.Generator().manual_seed(3)
    xb = torch.randn(T, D + 24, generator=g).cuda()
    lb = torch.zeros(T, E + 9, device="cuda")
    lb[:, 3:E + 3] = spread_logits(T, E).cuda()
    x, logits = xb[:, 7:D + 7], lb[:, 3:E + 3]
    y, tol = ref_moe(x, logits, w13, w2, topk)
    wide = torch.full((T + 2, D + 40), 2.0, device="cuda")
    fp4.moe(x, logits, w13, w2, topk, out=wide[1:T + 1, 8:D + 8])
    check_close(wide[1:T + 1, 8:D + 8], y, tol, torch.float32)
    assert (wide[0] == 2).all() and (wide[-1] == 2).all() and (wide[:, :8] == 2).all() and (wide[:, D + 8:] == 2).all()
    base = torch.randn(T, D, generator=g)
    acc = base.cuda()
    fp4.moe(x, logits, w13, w2, topk, out=acc, accumulate=True)
    check_close(acc, y + base.double(), tol + 2 * E24 * (y.abs() + base.abs().double()), torch.float32)
    assert fp4.moe(x[:0], logits[:0], w13, w2, topk).shape == (0, D)


def test_the_same_bits_every_time_on_any_stream_and_in_a_graph():
    T, E, D, I, topk = 9, 48, 1024, 256, 6
    w13, w2 = experts(E, D, I, 9)
    g = torch.Generator().manual_seed(4)
    x, logits = torch.randn(T, D, generator=g).cuda(), torch.randn(T, E, generator=g).cuda()
    other = [torch.randn(T, D, generator=g).cuda(), torch.randn(T, E, generator=g).cuda()]
    want, want2 = fp4.moe(x, logits, w13, w2, topk), fp4.moe(*other, w13, w2, topk)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(fp4.moe(*([x, logits] if i % 3 else other), w13, w2, topk))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want if i % 3 else want2) for i, v in enumerate(got))
    xs, ls = x.clone(), logits.clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = fp4.moe(xs, ls, w13, w2, topk)
            y = fp4.moe(xs, ls, w13, w2, topk, out=y, accumulate=True)
        graphs.append((gr, y))
    for gr, y in graphs * 2:
        y.zero_()
        gr.replay()
        assert torch.equal(y, want + want)
    xs.copy_(other[0]), ls.copy_(other[1])
    graphs[1][0].replay()
    assert torch.equal(graphs[1][1], want2 + want2)
    fp4.check()


def test_a_decode_step_of_the_operators_together():
    """Weights quantised on the device, a 4-bit projection, the expert layer on its output and a projection back."""
    T, H, E, D, I, topk = 4, 320, 24, 640, 128, 3
    g = torch.Generator().manual_seed(12)
    w_in = fp4.quantize((torch.randn(D, H, generator=g) * H ** -0.5).cuda(), "nvfp4", float(torch.tensor(0.01)))
    w_router = torch.randn(E, D, generator=g).cuda()
    w13, w2 = experts(E, D, I, 13)
    w_out = fp4.quantize((torch.randn(H, D, generator=g) * D ** -0.5).cuda(), "mxfp4")
    x = torch.randn(T, H, generator=g).cuda()
    a = fp4.linear(x, w_in)
    logits = a @ w_router.t()
    m = fp4.moe(a, logits, w13, w2, topk, scale=1.5, limit=10.0)
    y = fp4.linear(m, w_out, out_dtype=torch.bfloat16)
    fp4.check()
    xq, xin = fp4.reference_dequantize(fp4.quantize(x, "nvfp4")), fp4.reference_dequantize(w_in)
    want = xq @ xin.t()
    assert ((a.double() - want).abs() <= (H + 2) * E24 * (xq.abs() @ xin.abs().t())).all()
    check_close(m, *ref_moe(a, logits, w13, w2, topk, scale=1.5, limit=10.0), torch.float32)
    mq, wo = fp4.reference_dequantize(fp4.quantize(m)), fp4.reference_dequantize(w_out)
    want = mq @ wo.t()
    assert ((y.double() - want).abs() <= (D + 2) * E24 * (mq.abs() @ wo.abs().t()) + 2.0 ** -8 * want.abs()).all()


@pytest.mark.parametrize("rows", [1, 5])
def test_dsv41_decode_through_the_two_kernel_layer(rows):
    """The tiny DSV41 model with its routed experts as this layer against the per-pair expert kernels: both multiply the
    same e2m1 x e4m3 values, so the logits agree up to summation order; and a captured step replays it."""
    from ferrite_b200.models.dsv41 import DictWeights, Dsv41DeviceModel
    from ferrite_b200.models.dsv41_config import Dsv41Config
    from ferrite_b200.models.dsv41_weights import random_weights
    from ferrite_b200.utils.switches import Switches, set_switches
    cfg = Dsv41Config.tiny()
    w = random_weights(cfg, 4)
    ids = torch.randint(0, cfg.vocab_size - 20, (20,), generator=torch.Generator().manual_seed(3)).tolist()
    logits = {}
    try:
        for two in (False, True):
            set_switches(Switches(d4_moe_two=two))
            dev = Dsv41DeviceModel(cfg, DictWeights(w), max_rows=8, max_ctx=128)
            assert all(L["moe2"] == two for L in dev.layers)
            out = []
            for i in range(0, len(ids), rows):
                c = ids[i:i + rows]
                dev.forward(dev.make_rows([0], [len(c)]), torch.tensor(c, dtype=torch.int32, device="cuda"))
                out.append(dev.ws["logits"][:len(c)].cpu().clone())
            torch.cuda.synchronize()
            fp4.check()
            logits[two] = torch.cat(out)
            if two:
                rs = dev.make_rows([0], [1])
                tok = torch.tensor(ids[:1], dtype=torch.int32, device="cuda")
                dev.reset_slot(0)
                dev.forward(rs, tok, advance=False)
                want = dev.ws["logits"][:1].clone()
                dev.reset_slot(0)
                gr = torch.cuda.CUDAGraph()
                with torch.cuda.graph(gr):
                    dev.forward(rs, tok, advance=False)
                dev.ws["logits"].zero_()
                gr.replay()
                assert torch.equal(dev.ws["logits"][:1], want)
    finally:
        set_switches(None)
    a, b = logits[True], logits[False]
    assert (a - b).abs().max().item() < 2e-3 * b.abs().max().item(), (a - b).abs().max().item()
    assert torch.equal(a.argmax(-1), b.argmax(-1))


def test_in_place_and_nan_stays_in_its_rows():
    """out may be x; a token with a NaN, and an expert with a NaN scale in w13, reach the rows that have them only."""
    T, E, topk, D, I = 6, 8, 2, 256, 64
    w13, w2 = experts(E, D, I, 5)
    logits = spread_logits(T, E, 5).cuda()
    x = torch.randn(T, D, generator=torch.Generator().manual_seed(5)).cuda()
    want = fp4.moe(x, logits, w13, w2, topk)
    y = x.clone()
    fp4.moe(y, logits, w13, w2, topk, out=y)
    assert torch.equal(y, want)
    bad = x.clone()
    bad[2, 17] = float("nan")
    y = fp4.moe(bad, logits, w13, w2, topk)
    rest = [t for t in range(T) if t != 2]
    assert y[2].isnan().all() and torch.equal(y[rest], want[rest])
    chosen = logits.topk(topk).indices == int(logits[0].argmax())
    rows = chosen.any(1).cpu()
    assert rows.any() and not rows.all()
    broken = fp4.Fp4Tensor(w13.codes, w13.scales.clone(), "mxfp4", w13.shape)
    broken.scales[int(logits[0].argmax()), 0, 0, 0, 0] = 255     # gate, row 0, block 0
    y = fp4.moe(x, logits, broken, w2, topk)
    assert y[rows].isnan().all() and torch.equal(y[~rows], want[~rows])
    fp4.check()


@pytest.mark.parametrize("T", [1, 4, 24])
def test_a_chain_of_calls_that_each_read_what_the_one_before_wrote(T):
    """Kernels start beside the end of their predecessors: back to back, replayed from a graph, or with a wait after every
    call, the bits are the same."""
    D, E, topk, I = 1024, 8, 2, 256
    w13, w2 = experts(E, D, I, 7)
    g = torch.Generator().manual_seed(7)
    wa, wb = (fp4.quantize((torch.randn(D, D, generator=g) * D ** -0.5).cuda(), f) for f in ("nvfp4", "mxfp4"))
    x0 = torch.randn(T, D, generator=g).cuda()
    router = (torch.randn(E, D, generator=g) * D ** -0.5).cuda()

    def chain(after=lambda: None):
        x, seen = x0, []
        for _ in range(6):
            y = fp4.linear(x, wa)
            after()
            q = fp4.quantize(y, "mxfp4")
            after()
            z = fp4.dequantize(q, torch.float32)
            after()
            m = fp4.matmul(fp4.quantize(z, "mxfp4"), wb, torch.float32)
            after()
            m2 = fp4.matmul(q, wb, torch.float32, out=z)       # into what the quantiser before has just read
            after()
            x = fp4.moe(m, m2 @ router.t(), w13, w2, topk, scale=3.0, out=m2, accumulate=True)
            after()
            x = fp4.linear(x, wb)
            seen += [y, m, x]
            x = x / x.std()
            after()
        return seen

    want = chain(torch.cuda.synchronize)
    assert all(t.isfinite().all() and t.std() > 1e-3 for t in want)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(chain(), want))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = chain()
    for _ in range(5):
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    fp4.check()
