"""GPU: block-scaled 4-bit quantiser, expander and products (ops/fp4.py) against plain statements in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from ferrite_b200.ops import fp4  # noqa: E402
from ferrite_b200.ops import quant as Q  # noqa: E402

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def ref_values(x, fmt, ts=None):
    """Values (f64, CPU) that quantised x stands for, by the definition; a block that is not finite reads NaN."""
    u = x.float().cpu()
    if ts is not None:
        u = u / torch.tensor(ts, dtype=torch.float32)
    b = fp4.BLOCK[fmt]
    k = u.shape[-1]
    v = torch.nn.functional.pad(u, (0, -k % b)).unflatten(-1, (-1, b))
    amax = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    if fmt == "mxfp4":
        s = Q.pow2_ceil(amax.clamp_min(6 * 2.0 ** -126) * Q._INV6)
    else:
        s = Q.e4m3_round(amax.clamp_min(6 * 2.0 ** -9) / 6)
    y = Q.e2m1_decode(Q.e2m1_encode(v / s)).double() * s.double() * (1.0 if ts is None else ts)
    return torch.where(bad, torch.full((), math.nan, dtype=torch.float64), y).flatten(-2)[..., :k]


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 17), (16, 1000), (127, 129), (128, 128), (130, 256), (257, 700)])
def test_quantize_is_the_definition(fmt, dtype, rows, cols):
    """Codes and scales bit for bit: every value of the result is the definition's."""
    x = (torch.randn(rows, cols, generator=_gen(rows * 7 + cols)) * torch.logspace(-4, 3, rows).unsqueeze(1)).to(dtype)
    q = fp4.quantize(x.cuda(), fmt)
    assert same(fp4.reference_dequantize(q).cpu(), ref_values(x, fmt))
    tail = Q.e2m1_unpack(q.codes)[..., cols:]
    assert (tail & 7 == 0).all()                       # zero codes behind the last column
    pad = fp4.unpack_scales(q.scales, q.scales.shape[-3] * 128, q.scales.shape[-2] * 4)
    assert (pad[rows:] == 0).all() and (pad[:, -(-cols // fp4.BLOCK[fmt]):] == 0).all()


def test_quantize_bytes_are_the_checkpoint_codec_s():
    x = torch.randn(300, 320, generator=_gen(4)) * 0.05
    packed, scale = Q.quant_fp4_weight(x)
    q, want = fp4.quantize(x.cuda()), fp4.Fp4Tensor.from_rows(packed.cuda(), scale.cuda())
    assert torch.equal(q.scales, want.scales)
    zero = lambda c: torch.where(c & 7 == 0, 0, c)      # the sign of a zero is not part of the format's value
    assert torch.equal(zero(Q.e2m1_unpack(q.codes)), zero(Q.e2m1_unpack(want.codes)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_border_of_two_codes(dtype):
    """Values exactly on, and one ulp to either side of, every border between codes, under many e4m3 scales."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    scales = torch.arange(0x18, 0x60, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    v = scales[:, None] * mids[None, :]
    up, dn = torch.nextafter(v, torch.tensor(math.inf)), torch.nextafter(v, torch.tensor(0.0))
    x = torch.cat([v, -v], 1)
    y = torch.cat([up, dn], 1) if dtype == torch.float32 else x.flip(1)
    top = scales[:, None] * 6
    rows = torch.cat([torch.cat([x, top, x[:, :1]], 1), torch.cat([y, top, x[:, :1]], 1)], 0).to(dtype)
    assert rows.shape[1] == 16
    for fmt in ("nvfp4", "mxfp4"):
        assert same(fp4.reference_dequantize(fp4.quantize(rows.cuda(), fmt)).cpu(), ref_values(rows, fmt))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quotients_by_every_e4m3_scale(dtype):
    """Every scale byte (its block holds 6 s), with values at random and a few steps around every border of two codes."""
    g = _gen(11)
    s = torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()[:, None, None]
    x = torch.empty(126, 64, 16)
    near = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])[torch.randint(0, 7, (126, 32, 16), generator=g)] * s
    bits = near.view(torch.int32) + torch.randint(-3, 4, near.shape, generator=g, dtype=torch.int32)
    x[:, :32] = bits.view(torch.float32) * (1 - 2 * torch.randint(0, 2, near.shape, generator=g))
    x[:, 32:] = (torch.rand(126, 32, 16, generator=g) * 2 - 1) * 6 * s
    x[:, :, 3] = 6 * s[:, :, 0]
    x = x.view(126, 1024).to(dtype)
    q = fp4.quantize(x.cuda(), "nvfp4")
    assert same(fp4.reference_dequantize(q).cpu(), ref_values(x, "nvfp4"))
    assert torch.equal(fp4.unpack_scales(q.scales, 126, 64).cpu(), torch.arange(1, 127, dtype=torch.uint8)[:, None].expand(126, 64))


@pytest.mark.parametrize("ts", [1.0, 0.00037, 2.0 ** -20, 3.7e5, 2.0 ** -100, 2.0 ** 100])
def test_tensor_scale(ts):
    ts = float(torch.tensor(ts))
    x = torch.randn(130, 144, generator=_gen(3)) * ts * 100
    q = fp4.quantize(x.cuda(), "nvfp4", tensor_scale=ts)
    assert same(fp4.reference_dequantize(q).cpu(), ref_values(x, "nvfp4", ts))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_values_that_are_not_finite_and_extremes(fmt):
    x = torch.randn(8, 256, generator=_gen(1))
    x[0, 5], x[1, 40], x[2, 200], x[3] = math.nan, math.inf, -math.inf, 0.0
    x[4], x[5], x[6, 0] = 1e-44, 3.4028234e38, -3.4028234e38
    q = fp4.quantize(x.cuda(), fmt)
    got, want = fp4.reference_dequantize(q).cpu(), ref_values(x, fmt)
    assert same(got, want) and torch.isnan(got[0]).sum() == fp4.BLOCK[fmt]
    d = fp4.dequantize(q, torch.float32).cpu()
    assert same(d.double(), want.float().double())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_rounds_once(fmt, dtype):
    ts = None if fmt == "mxfp4" else float(torch.tensor(0.0123))
    x = torch.randn(2, 131, 203, generator=_gen(9))
    q = fp4.quantize(x.cuda(), fmt, ts)
    f32 = fp4.reference_dequantize(fp4.Fp4Tensor(q.codes, q.scales, fmt, q.shape)).float()   # exact: 2 x 4 bits
    want = (f32 * (1.0 if ts is None else ts)).to(dtype)
    assert torch.equal(fp4.dequantize(q, dtype), want)
    wide = torch.full((2, 131, 301), 7.0, dtype=dtype, device="cuda")
    fp4.dequantize(q, out=wide[..., 50:253])
    assert torch.equal(wide[..., 50:253], want) and (wide[..., :50] == 7).all() and (wide[..., 253:] == 7).all()


def test_strided_and_batched_inputs():
    base = torch.randn(5, 40, 100, generator=_gen(2)).cuda()
    for x in (base[:, :, 3:90], base[1:4, ::2, :64], base[2, :, 1:], base[:, 4:5, :33]):
        q, c = fp4.quantize(x, "nvfp4"), fp4.quantize(x.contiguous(), "nvfp4")
        assert torch.equal(q.codes, c.codes) and torch.equal(q.scales, c.scales)


def ref_matmul(a, b):
    """Product in 64 bits and the sum of absolute products (what an f32 accumulation's error is relative to)."""
    A, B = fp4.reference_dequantize(a), fp4.reference_dequantize(b)
    return A @ B.t(), A.abs() @ B.abs().t()


def close(got, want, mag, K, dtype):
    """f32 accumulation of K products in any order: K half steps of f32 of the absolute sum; then one rounding."""
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    # f16 results below its normal range: half a subnormal step
    tol = (K + 2) * 2.0 ** -24 * mag + eps * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 256), (2, 130, 64), (16, 127, 1000), (17, 300, 96), (33, 129, 2048),
                                   (65, 257, 33), (100, 512, 4160), (128, 128, 128), (129, 255, 160), (333, 1111, 1000),
                                   (300, 640, 4096), (1, 5120, 8192), (1000, 4700, 1000), (1024, 4608, 640), (1200, 4609, 160),
                                   (2304, 8200, 96)])
def test_matmul(fmt, M, N, K):
    g = _gen(M + N + K)
    a = fp4.quantize((torch.randn(M, K, generator=g) * torch.rand(M, 1, generator=g) * 3).cuda(), fmt)
    b = fp4.quantize(torch.randn(N, K, generator=g).cuda(), fmt)
    want, mag = ref_matmul(a, b)
    for dtype in DTYPES:
        y = fp4.matmul(a, b, dtype)
        fp4.check()
        close(y, want, mag, K, dtype)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_every_scale_and_code_position_of_a_tile(fmt):
    """One row of ones against weights whose every block has its own scale and every column its own code."""
    N, K = 256, 512
    g = _gen(0)
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=g)
    lo, hi = (118, 136) if fmt == "mxfp4" else (0x20, 0x60)
    scale = torch.randint(lo, hi, (N, K // fp4.BLOCK[fmt]), dtype=torch.uint8, generator=g)
    w = fp4.Fp4Tensor.from_rows(codes.cuda(), scale.cuda(), fmt)
    for rows in (K, 200):   # one-hot rows: both operand orders
        x = fp4.quantize(torch.eye(K)[:rows].cuda(), fmt)
        assert torch.equal(fp4.matmul(x, w, torch.float32).double(),
                           fp4.reference_dequantize(x) @ fp4.reference_dequantize(w).t())
    x = fp4.quantize(torch.eye(K)[:100].cuda(), fmt)
    assert torch.equal(fp4.matmul(x, w, torch.float32).double(), fp4.reference_dequantize(x) @ fp4.reference_dequantize(w).t())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_nan_scales_reach_their_rows_only(fmt):
    x = torch.randn(200, 512, generator=_gen(6))
    x[7, 300] = math.nan
    w = torch.randn(140, 512, generator=_gen(7))
    w[3, 0] = math.inf
    for m in (200, 20):
        y = fp4.matmul(fp4.quantize(x[:m].cuda(), fmt), fp4.quantize(w.cuda(), fmt), torch.float32).cpu()
        bad = torch.isnan(y)
        want = torch.zeros(m, 140, dtype=torch.bool)
        want[7], want[:, 3] = True, True
        assert torch.equal(bad, want)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N,K", [(1, 384, 1000), (1, 5120, 8192), (2, 640, 2000), (5, 130, 700), (16, 257, 96), (1, 64, 1), (9, 256, 4096),
                                   (40, 200, 640), (200, 300, 384)])
def test_linear_is_quantize_and_matmul(fmt, M, N, K):
    g = _gen(K)
    ts = float(torch.tensor(0.03)) if fmt == "nvfp4" else None
    w = fp4.quantize(torch.randn(N, K, generator=g).cuda(), fmt, ts)
    for dtype in DTYPES:
        x = torch.randn(M, K + 8, generator=g).to(dtype).cuda()[:, 8:]
        want = fp4.matmul(fp4.quantize(x, fmt, ts), w, dtype)
        assert torch.equal(fp4.linear(x, w, x_scale=ts), want)
        wide = torch.full((M, N + 24), 3.0, dtype=dtype, device="cuda")
        fp4.linear(x, w, out=wide[:, 5:N + 5], x_scale=ts)
        assert torch.equal(wide[:, 5:N + 5], want) and (wide[:, :5] == 3).all() and (wide[:, N + 5:] == 3).all()
    fp4.check()


def test_the_same_bits_every_time_on_any_stream_and_in_a_graph():
    g = _gen(11)
    w = fp4.quantize(torch.randn(1280, 4096, generator=g).cuda(), "nvfp4")
    xs = [torch.randn(m, 4096, generator=g).cuda().bfloat16() for m in (1, 16, 100, 300)]
    want = [fp4.linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(fp4.linear(xs[i % 4], w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(got))
    x = xs[1].clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = fp4.linear(x, w)
        graphs.append((gr, y))
    for gr, y in graphs * 2:
        y.zero_()
        gr.replay()
        assert torch.equal(y, want[1])
    x.copy_(torch.randn(16, 4096, generator=g))
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], fp4.linear(x, w))
    fp4.check()


def test_empty_rows():
    w = fp4.quantize(torch.randn(64, 256).cuda())
    assert fp4.linear(torch.empty(0, 256, device="cuda"), w).shape == (0, 64)
    e = fp4.quantize(torch.empty(0, 256, device="cuda"))
    assert fp4.matmul(e, w).shape == (0, 64) and fp4.dequantize(e).shape == (0, 256)
    assert fp4.matmul(w, e).shape == (64, 0)
    assert fp4.quantize(torch.empty(0, 4, 64, device="cuda")).shape == (0, 4, 64)


def test_columns_of_one_buffer_and_interleaved_batches():
    """x and out beside each other in one buffer; an out whose matrices interleave."""
    w = fp4.quantize(torch.randn(96, 256).cuda())
    b = torch.randn(5, 400, device="cuda")
    want = fp4.linear(b[:, :256].clone(), w)
    fp4.linear(b[:, :256], w, out=b[:, 300:396])
    assert torch.equal(b[:, 300:396], want)
    q = fp4.quantize(torch.randn(3, 40, 72).cuda())
    o = torch.empty(40, 3, 72, device="cuda").transpose(0, 1)
    assert torch.equal(fp4.dequantize(q, out=o), fp4.dequantize(q, torch.float32))


FIRST_IN_CAPTURE = """
import torch
from ferrite_b200.ops import fp4
x = torch.randn({M}, 512, device="cuda").bfloat16()
wf = torch.randn(384, 512, device="cuda")
logits = torch.randn({M}, 4, device="cuda")
codes = lambda *s: torch.randint(0, 256, s, dtype=torch.uint8, device="cuda")
w13 = fp4.Fp4Tensor(codes(4, 2, 128, 256), torch.full((4, 2, 1, 4, 512), 120, dtype=torch.uint8, device="cuda"), "mxfp4", (4, 2, 128, 512))
w2 = fp4.Fp4Tensor(codes(4, 512, 64), torch.full((4, 4, 1, 512), 120, dtype=torch.uint8, device="cuda"), "mxfp4", (4, 512, 128))
def run():
    w = fp4.quantize(wf, "nvfp4")
    y = fp4.linear(x, w)
    return w.codes, y, fp4.matmul(fp4.quantize(x, "nvfp4"), w), fp4.moe(x, logits, w13, w2, 2)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
fp4.check()
"""


@pytest.mark.parametrize("M", [1, 20])
def test_the_first_call_of_a_process_may_be_captured(M):
    import os
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE.format(M=M)], cwd=root, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": root})
    assert r.returncode == 0, r.stderr[-3000:]


def test_two_threads_on_two_streams():
    import threading
    w = fp4.quantize(torch.randn(512, 1024).cuda())
    xs = [torch.randn(m, 1024, device="cuda") for m in (1, 7)]
    want = [fp4.linear(x, w) for x in xs]
    got = [[], []]

    def work(i):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(st):
            got[i] += [fp4.linear(xs[i], w) for _ in range(20)]
        st.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(len(got[i]) == 20 and all(torch.equal(y, want[i]) for y in got[i]) for i in (0, 1))
    fp4.check()


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 values: the last rows are what they are in a small call."""
    R, C = 300_000, 8192
    t0 = R // 128 * 128
    x = torch.empty(R, C, dtype=torch.bfloat16, device="cuda")
    x[:t0].fill_(1.0)
    x[t0:] = torch.randn(R - t0, C, generator=_gen(4)).cuda()
    for fmt in ("mxfp4", "nvfp4"):
        q, tail = fp4.quantize(x, fmt), fp4.quantize(x[t0:], fmt)
        assert torch.equal(q.codes[t0:], tail.codes) and torch.equal(q.scales[t0 // 128:], tail.scales)
        d = fp4.dequantize(q)
        assert torch.equal(d[t0:], fp4.dequantize(tail)) and torch.equal(d[:4], fp4.dequantize(fp4.quantize(x[:4], fmt)))
        del q, d
    w = fp4.quantize(torch.randn(C, 128, generator=_gen(5)).cuda(), "nvfp4")
    xs = x[:, :128]
    y = fp4.linear(xs, w)
    assert y.numel() > 2 ** 31
    for rows in (slice(0, 256), slice(t0, R)):
        assert torch.equal(y[rows], fp4.linear(xs[rows].contiguous(), w))
    fp4.check()


def test_a_tensor_scale_is_multiplied_in_f32_before_the_rounding_to_16_bits():
    """A value whose product with the scale lies 2e-6 of a step below the middle of two bf16: its f32 rounding is the middle,
    which goes to the even neighbour above.  (Rounded once it would be the one below.)"""
    ts, v = 0.04430042579770088, 0.0859375
    assert float(torch.tensor(ts)) == ts
    scale = torch.zeros(1, 1, 1, 512, dtype=torch.uint8)
    scale[..., 0] = torch.tensor(v * 2).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.zeros(1, 64, dtype=torch.uint8)
    codes[0, 0] = 1                                                                     # 0.5
    q = fp4.Fp4Tensor(codes.cuda(), torch.cat([scale, torch.zeros_like(scale)], 2)[0].cuda(), "nvfp4", (1, 16), ts)
    assert float(fp4.reference_dequantize(q)[0, 0]) == v * ts
    assert float(fp4.dequantize(q, torch.float32)[0, 0]) == float(torch.tensor(v) * torch.tensor(ts))
    below, above = 0.0037994384765625, 0.003814697265625
    assert v * ts < (below + above) / 2 and float(fp4.dequantize(q)[0, 0]) == above
