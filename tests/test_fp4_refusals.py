"""CPU: what the 4-bit operators refuse, and the layout of their scale chunks."""
import pytest
import torch

from ferrite_b200.ops import fp4
from ferrite_b200.ops import quant as Q


def test_scale_chunks_round_trip_and_place():
    s = torch.randint(0, 255, (3, 200, 7), dtype=torch.uint8)
    c = fp4.pack_scales(s)
    assert c.shape == (3, 2, 2, 512)
    assert torch.equal(fp4.unpack_scales(c, 200, 7), s)
    for r, b in ((0, 0), (33, 5), (127, 3), (199, 6)):
        assert c[1, r // 128, b // 4, r % 32 * 16 + r % 128 // 32 * 4 + b % 4] == s[1, r, b]


def test_from_rows_is_the_checkpoint_codec():
    w = torch.randn(130, 192)
    packed, scale = Q.quant_fp4_weight(w)
    t = fp4.Fp4Tensor.from_rows(packed, scale)
    assert t.codes.shape == (130, 128) and (t.codes[:, 96:] == 0).all()
    assert torch.equal(fp4.reference_dequantize(t).float(), Q.dequant_fp4_weight(packed, scale))


def _t(rows=4, cols=64, fmt="mxfp4", lead=()):
    g = (cols + 127) // 128
    c = g if fmt == "mxfp4" else 2 * g
    return fp4.Fp4Tensor(torch.zeros(*lead, rows, 64 * g, dtype=torch.uint8),
                         torch.zeros(*lead, (rows + 127) // 128, c, 512, dtype=torch.uint8), fmt, (*lead, rows, cols))


def test_a_tensor_s_parts_have_to_belong_together():
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8)
    fp4.Fp4Tensor(codes, scales, "mxfp4", (4, 128))
    for bad in [(codes, scales, "mxfp8", (4, 128)), (codes, scales, "mxfp4", (4, 129)), (codes, scales, "nvfp4", (4, 128)),
                (codes, scales, "mxfp4", (128,)), (codes, scales, "mxfp4", (4, 0)), (codes[:3], scales, "mxfp4", (4, 128)),
                (codes, scales, "mxfp4", (4, 128), 2.0)]:
        with pytest.raises(ValueError):
            fp4.Fp4Tensor(*bad)
    with pytest.raises(TypeError):
        fp4.Fp4Tensor(codes.int(), scales, "mxfp4", (4, 128))
    with pytest.raises(ValueError):   # not contiguous
        fp4.Fp4Tensor(torch.zeros(4, 128, dtype=torch.uint8)[:, ::2], scales, "mxfp4", (4, 128))
    with pytest.raises(ValueError):   # not aligned
        fp4.Fp4Tensor(torch.zeros(257, dtype=torch.uint8)[1:].view(4, 64), scales, "mxfp4", (4, 128))


def test_refusals_before_any_launch():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        fp4.quantize(x)
    with pytest.raises(ValueError, match="fmt"):
        fp4.quantize(x, "int4")
    with pytest.raises(TypeError):
        fp4.quantize(x.double())
    for ts in (0.0, -1.0, float("nan"), float("inf"), 2.0 ** -101, "1"):
        with pytest.raises(ValueError, match="tensor_scale"):
            fp4.quantize(x, "nvfp4", tensor_scale=ts)
    with pytest.raises(ValueError, match="nvfp4"):
        fp4.quantize(x, "mxfp4", tensor_scale=1.0)
    with pytest.raises(ValueError, match="CUDA"):
        fp4.dequantize(_t())
    with pytest.raises(ValueError, match=r"\[M, K\]"):
        fp4.matmul(_t(4, 64), _t(4, 96))
    with pytest.raises(ValueError, match="one format"):
        fp4.matmul(_t(4, 64), _t(4, 64, "nvfp4"))
    with pytest.raises(ValueError, match="CUDA"):
        fp4.matmul(_t(), _t())
    with pytest.raises(ValueError, match=r"\[M, K\]"):
        fp4.linear(torch.zeros(2, 4, 64), _t())
    with pytest.raises(ValueError, match="CUDA"):
        fp4.linear(x, _t())


@pytest.mark.parametrize("x", [torch.zeros(4, 64).t(), torch.zeros(4, 64)[:, ::2], torch.zeros(1, 64).expand(4, 64),
                               torch.zeros(64), torch.zeros(4, 0)])
def test_layouts_that_are_refused(x, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    with pytest.raises(ValueError):
        fp4._matrix(x, "x")


def test_layouts_that_are_taken(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    b = torch.zeros(6, 5, 40, 100)
    assert fp4._matrix(b, "x") == (30, 40, 100, 4000, 100)
    assert fp4._matrix(b[:, :, :8, :60], "x") == (30, 8, 60, 4000, 100)
    assert fp4._matrix(b[2:3, 1:2], "x")[:3] == (1, 40, 100)
    assert fp4._matrix(b[:, 2], "x") == (6, 40, 100, 20000, 100)
    with pytest.raises(ValueError, match="common stride"):
        fp4._matrix(b[:, :3], "x")


def _moe_args(T=2, E=4, I=64, D=128):
    return [torch.zeros(T, D), torch.zeros(T, E), _t(I, D, lead=(E, 2)), _t(D, I, lead=(E,)), 2]


@pytest.mark.parametrize("change,match", [
    (lambda a, k: k.update(score="tanh"), "score"),
    (lambda a, k: a.__setitem__(2, _t(64, 128, "nvfp4", (4, 2))), "mxfp4"),
    (lambda a, k: a.__setitem__(2, _t(64, 128, lead=(4,))), "w13"),
    (lambda a, k: a.__setitem__(3, _t(64, 128, lead=(4,))), "w2"),
    (lambda a, k: a.__setitem__(0, torch.zeros(2, 127)), r"\[T, 128\]"),
    (lambda a, k: a.__setitem__(4, 5), "topk"),
    (lambda a, k: a.__setitem__(4, 0), "topk"),
    (lambda a, k: a.__setitem__(1, torch.zeros(2, 5)), "logits"),
    (lambda a, k: a.__setitem__(1, torch.zeros(2, 4).bfloat16()), "logits"),
    (lambda a, k: a.__setitem__(1, torch.zeros(4, 2).t()), "logits"),
    (lambda a, k: k.update(bias=torch.zeros(3)), "bias"),
    (lambda a, k: k.update(limit=-1.0), "limit"),
    (lambda a, k: k.update(limit=float("nan")), "limit"),
    (lambda a, k: k.update(scale=float("inf")), "scale"),
    (lambda a, k: k.update(accumulate=True), "out"),
    (lambda a, k: None, "CUDA"),
])
def test_moe_refusals(change, match):
    a, k = _moe_args(), {}
    change(a, k)
    with pytest.raises(ValueError, match=match):
        fp4.moe(*a, **k)


def test_moe_limits():
    with pytest.raises(ValueError, match="32 tokens"):
        fp4.moe(*_moe_args(T=33))
    with pytest.raises(ValueError, match="multiple of 32"):
        fp4.moe(*_moe_args(I=48))
    with pytest.raises(ValueError, match="512 experts"):
        fp4.moe(*_moe_args(E=513, I=32, D=32))
    with pytest.raises(ValueError, match="up to 8192"):
        fp4.moe(*_moe_args(E=2, I=32, D=8193))


def test_overlap_of_out_and_x(monkeypatch):
    b = torch.zeros(4, 256)
    assert fp4._overlap(b, b[2:]) and fp4._overlap(b[:, :200], b[:, 100:]) and not fp4._overlap(b[:2], b[2:])
    assert not fp4._overlap(b[:0], b) and not fp4._overlap(b, torch.zeros(4))
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    with pytest.raises(ValueError, match="share memory"):
        fp4.linear(b[:1, :64], _t(64, 64), out=b[:1, :64])


def test_columns_of_one_buffer_beside_each_other():
    b = torch.zeros(4, 256)
    assert not fp4._overlap(b[:, :100], b[:, 100:]) and not fp4._overlap(b[:, 100:], b[:, :100])
    assert not fp4._overlap(b[2:, :100], b[:3, 100:]) and fp4._overlap(b[:, :101], b[:, 100:])
    assert not fp4._overlap(b[:, 100:], b[:, :100].view(torch.int32))
    assert fp4._overlap(b[:, :100], b.view(2, 512)[:, 100:])   # another row stride: the spans decide


def test_an_out_that_meets_itself_or_an_operand(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    q = _t(8, 64, lead=(3,))
    with pytest.raises(ValueError, match="matrices of out overlap"):
        fp4.dequantize(q, out=torch.zeros(8, 64).expand(3, 8, 64))
    with pytest.raises(ValueError, match="matrices of out overlap"):
        fp4.dequantize(q, out=torch.zeros(4096).as_strided((3, 8, 64), (65, 128, 1)))
    for out in (torch.zeros(8, 3, 64).transpose(0, 1), torch.zeros(3, 8, 100)[:, :, :64]):   # these do not
        assert fp4._out(out, (3, 8, 64), out.dtype, out.device)[0] is out
    w = _t(4, 64)
    with pytest.raises(ValueError, match="share memory"):
        fp4.matmul(_t(8, 64), w, out=w.codes.view(-1)[:128].view(torch.float32).view(8, 4))


def test_tensor_scales_whose_product_leaves_f32(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    for xs, ws in ((2.0 ** 80, 2.0 ** 80), (2.0 ** -80, 2.0 ** -80)):
        w = _t(4, 64, "nvfp4")
        w.tensor_scale = ws
        x = _t(4, 64, "nvfp4")
        x.tensor_scale = xs
        with pytest.raises(ValueError, match="product of the tensor scales"):
            fp4.matmul(x, w)
        with pytest.raises(ValueError, match="product of the tensor scales"):
            fp4.linear(torch.zeros(4, 64), w, x_scale=xs)


def test_from_rows_refusals():
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    for packed, scale in ((z(16), z(1)), (z(4, 0), z(4, 0)), (z(4, 16), z(4, 2)), (z(4, 8), z(4, 1))):
        with pytest.raises(ValueError):
            fp4.Fp4Tensor.from_rows(packed, scale)


def test_from_rows_copies_bytes_on_any_boundary():
    raw = torch.randint(0, 256, (3 + 4 * 64,), dtype=torch.uint8)
    packed = raw[3:].view(4, 64)
    t = fp4.Fp4Tensor.from_rows(packed, torch.zeros(4, 4, dtype=torch.uint8))
    before = t.codes.clone()
    raw.zero_()
    assert torch.equal(t.codes, before) and before.any()
    u = t.to("cpu")
    assert u.shape == t.shape and torch.equal(u.codes, t.codes) and torch.equal(u.scales, t.scales)


@pytest.mark.parametrize("status", [torch.zeros(4), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32),
                                    torch.zeros(8, dtype=torch.int32)[::2], torch.zeros(4, dtype=torch.int32, device="meta")])
def test_status_words_that_are_refused(status, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    for call in (lambda: fp4.matmul(_t(4, 64), _t(8, 64), status=status), lambda: fp4.linear(torch.zeros(4, 64), _t(8, 64), status=status),
                 lambda: fp4.moe(*_moe_args(), status=status)):
        with pytest.raises(ValueError, match="status must be"):
            call()


def test_status_words_reach_the_kernels(monkeypatch):
    """A given tensor, or nothing, is what the entry point is handed behind its last number."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    seen = []
    monkeypatch.setattr(fp4, "_call", lambda device, name, *args: seen.append((name, args[-1])))
    own = torch.zeros(12, dtype=torch.int32)[4:8]
    for status in (own, None):
        fp4.matmul(_t(4, 64), _t(8, 64), status=status)
        fp4.linear(torch.zeros(4, 64), _t(8, 64), status=status)
        fp4.moe(*_moe_args(), status=status)
    assert [n for n, _ in seen] == ["fb_fp4_matmul", "fb_fp4_linear", "fb_fp4_moe"] * 2
    assert all(s is own for _, s in seen[:3]) and all(s is None for _, s in seen[3:])


@pytest.mark.parametrize("scale", [1e39, -1e39, float("nan"), float("-inf")])
def test_a_scale_that_f32_does_not_hold(scale):
    with pytest.raises(ValueError, match="finite"):
        fp4.moe(*_moe_args(), scale=scale)
