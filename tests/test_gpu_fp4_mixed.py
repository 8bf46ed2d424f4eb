"""GPU: 4-bit operators next to the framework's other kernels."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from ferrite_b200 import _lib  # noqa: E402
from ferrite_b200.ops import fp4  # noqa: E402


def test_expanded_weights_of_a_gemv_with_early_starts():
    """A decode GEMV reads the weights that the expander before it wrote, with every kernel allowed to start early."""
    N, D, m = 4096, 4096, 2
    K = _lib.lib()
    g = torch.Generator().manual_seed(6)
    q = fp4.quantize((torch.randn(N, D, generator=g) * 0.1).cuda(), "nvfp4")
    xs = torch.zeros(4, m, D, dtype=torch.int16, device="cuda")
    K.call("fb_split_rows", torch.randn(m, D, generator=g).cuda(), D, xs, D, m * D, 3, m, D)
    w, out = torch.empty(N, D, dtype=torch.bfloat16, device="cuda"), torch.empty(m, N, device="cuda")
    gemv = lambda: K.call("fb_gemv_mma_bf16", w, xs, D, m * D, out, N, m, N, D, 0, 0, None, 0, 0, 0)
    fp4.dequantize(q, out=w)
    torch.cuda.synchronize()
    gemv()
    torch.cuda.synchronize()
    want = out.clone()
    K.lib.fb_set_pdl(1)
    try:
        for _ in range(20):
            w.fill_(3.0), out.zero_()
            fp4.dequantize(q, out=w)
            gemv()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    finally:
        K.lib.fb_set_pdl(0)


def test_a_wait_that_ran_out_in_the_expert_layer_fails_the_engine_s_step(monkeypatch):
    """The report of an expired wait, put into the words that the expert layer was given (by the host: nothing hangs), raises on
    the step that caused it, and the next step is clean."""
    from ferrite_b200.engine.dsv41_engine import Dsv41Engine
    from ferrite_b200.models.dsv41 import DictWeights
    from ferrite_b200.models.dsv41_config import Dsv41Config
    from ferrite_b200.models.dsv41_weights import random_weights
    from ferrite_b200.parallel.status import CollectiveTimeout, FB_TIMEOUT
    from ferrite_b200.utils.switches import Switches, set_switches
    cfg = Dsv41Config.tiny()
    try:
        set_switches(Switches(d4_moe_two=True))
        eng = Dsv41Engine(cfg, DictWeights(random_weights(cfg, 4)), max_ctx=128, use_graphs=False)
        eng.prefill([5, 9, 2, 7])
        eng.step_plain()
        real, expired = fp4.moe, []

        def moe(*args, **kw):
            y = real(*args, **kw)
            if not expired:
                kw["status"][:4].copy_(torch.tensor([FB_TIMEOUT, 3, 1008, 2], dtype=torch.int32))
                expired.append(1)
            return y

        monkeypatch.setattr(fp4, "moe", moe)
        with pytest.raises(CollectiveTimeout):
            eng.step_plain()
        assert expired
        eng.step_plain()
    finally:
        set_switches(None)


def test_a_call_writes_no_status_when_nothing_ran_out():
    w = fp4.quantize(torch.randn(64, 256).cuda())
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.randn(3, 256).cuda()
    assert torch.equal(fp4.linear(x, w, status=status), fp4.linear(x, w))
    assert torch.equal(fp4.matmul(fp4.quantize(x), w, status=status), fp4.linear(x, w, out_dtype=torch.bfloat16))
    assert status.tolist() == [0, 0, 0, 0]


def test_what_the_expert_layer_keeps_twice_is_what_the_estimate_counts():
    from ferrite_b200.models.dsv41 import DictWeights, Dsv41DeviceModel
    from ferrite_b200.models.dsv41_config import Dsv41Config
    from ferrite_b200.models.dsv41_weights import moe_two_bytes, random_weights
    from ferrite_b200.utils.switches import Switches, set_switches
    cfg = Dsv41Config.tiny()
    try:
        set_switches(Switches(d4_moe_two=True))
        dev = Dsv41DeviceModel(cfg, DictWeights(random_weights(cfg, 4)), max_rows=8, max_ctx=128)
    finally:
        set_switches(None)
    kept = 0
    for L in dev.layers + [m for m in dev.mtp]:
        assert L["moe2"] and L["moe2_w13"].codes.data_ptr() == L["w13"].data_ptr()
        kept += L["moe2_w13"].scales.numel() + L["moe2_w2"].scales.numel()
        kept += L["moe2_w2"].codes.numel() if L["moe2_w2"].codes.data_ptr() != L["w2"].data_ptr() else 0
    assert kept == moe_two_bytes(cfg)


def test_the_words_of_check_are_clean_after_ordinary_calls():
    """Read without and with clearing them."""
    import ctypes
    w = fp4.quantize(torch.randn(64, 256).cuda())
    fp4.linear(torch.randn(3, 256).cuda(), w)
    host = (ctypes.c_int * 4)(7, 7, 7, 7)
    for clear in (0, 1):
        _lib.lib().call("fb_fp4_status", ctypes.cast(host, ctypes.POINTER(ctypes.c_int)), clear)
        assert list(host) == [0, 0, 0, 0]
    fp4.check()


@pytest.mark.parametrize("M,N,K", [(150, 1111, 96), (333, 1111, 1000), (700, 4097, 160), (1200, 4609, 160), (20, 1111, 96)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_outputs_that_end_inside_a_unit_of_an_aligned_buffer(M, N, K, dtype):
    """Rows that TMA can address (a 16-byte base and row stride) whose last column lies inside a 16-byte unit: what is behind it, and
    the rows around, stay as they were."""
    g = torch.Generator().manual_seed(N)
    a, b = fp4.quantize(torch.randn(M, K, generator=g).cuda(), "nvfp4"), fp4.quantize(torch.randn(N, K, generator=g).cuda(), "nvfp4")
    want = fp4.matmul(a, b, dtype)
    wide = torch.full((M + 2, -(-N // 8) * 8 + 24), 5.0, dtype=dtype, device="cuda")
    out = wide[1:M + 1, 8:N + 8]
    assert out.data_ptr() % 16 == 0 and out.stride(0) * out.element_size() % 16 == 0
    fp4.matmul(a, b, out=out)
    fp4.check()
    assert torch.equal(out, want)
    assert (wide[0] == 5).all() and (wide[-1] == 5).all() and (wide[:, :8] == 5).all() and (wide[:, N + 8:] == 5).all()


def test_a_matrix_times_itself():
    for n in (50, 300):
        q = fp4.quantize(torch.randn(n, 448, generator=torch.Generator().manual_seed(n)).cuda(), "mxfp4")
        y = fp4.matmul(q, q, torch.float32)
        v = fp4.reference_dequantize(q)
        assert ((y.double() - v @ v.t()).abs() <= 450 * 2.0 ** -24 * (v.abs() @ v.abs().t())).all()


def test_the_widest_routing_and_two_graphs_of_one_pool():
    """512 experts, 32 tokens with 32 experts each and a bias: the routing's scratch fills the stages; captured twice into one
    pool, replayed in turn."""
    from test_gpu_fp4_moe import check_close, experts, ref_moe, spread_logits
    T, E, D, I, topk = 32, 512, 256, 32, 32
    w13, w2 = experts(E, D, I, 31)
    g = torch.Generator().manual_seed(32)
    x, logits = torch.randn(T, D, generator=g).cuda(), spread_logits(T, E, 33).cuda()
    bias = (torch.randperm(E, generator=g).float() * 0.37 / E).cuda()
    want = fp4.moe(x, logits, w13, w2, topk, bias=bias)
    check_close(want, *ref_moe(x, logits, w13, w2, topk, bias=bias), torch.float32)
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            y = fp4.moe(x, logits, w13, w2, topk, bias=bias)
        graphs.append((gr, y))
    for gr, y in graphs * 3:
        y.zero_()
        gr.replay()
        assert torch.equal(y, want)
    fp4.check()


@pytest.mark.parametrize("T", [7, 8, 9, 31])
def test_the_same_token_many_times_gives_the_same_row(T):
    from test_gpu_fp4_moe import experts
    E, D, I, topk = 24, 640, 96, 5
    w13, w2 = experts(E, D, I, 41)
    g = torch.Generator().manual_seed(42)
    x, logits = torch.randn(1, D, generator=g).cuda(), torch.randn(1, E, generator=g).cuda()
    y = fp4.moe(x.repeat(T, 1), logits.repeat(T, 1), w13, w2, topk)
    assert torch.equal(y, y[:1].expand(T, D)) and y.abs().max() > 0.1


@pytest.mark.parametrize("captured", [False, True])
def test_operands_made_on_another_stream(captured):
    """Fork and join around every operator: one operand comes late from a second stream and the kernel before on the first one lets
    its dependents start early; what the second stream wrote is what is read."""
    from test_gpu_fp4_moe import experts
    T, E, D, I, topk = 4, 8, 1024, 128, 2
    g = torch.Generator().manual_seed(51)
    w13, w2 = experts(E, D, I, 52)
    w = fp4.quantize(torch.randn(1280, D, generator=g).cuda(), "nvfp4")
    big = torch.randn(4096, 4096, generator=g).cuda()
    xs = {m: torch.randn(m, D, generator=g).cuda() for m in (1, 20, 300)}
    x, logits = torch.randn(T, D, generator=g).cuda(), torch.randn(T, E, generator=g).cuda()
    bufs = {m: torch.empty_like(v) for m, v in xs.items()}
    xb, lb = torch.empty_like(x), torch.empty_like(logits)
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    small = torch.randn(64, 128, device="cuda")

    def late(dst, src):
        """On the other stream: some work, then dst = src."""
        side.wait_stream(main)
        with torch.cuda.stream(side):
            dst.fill_(7.0)
            a = big
            for _ in range(3):
                a = a @ big
            dst.copy_(src)
            dst.add_(a[:1, :1] * 0.0)
        fp4.quantize(small)                      # on the main stream, ends long before
        main.wait_stream(side)

    def run():
        out = []
        for m in xs:
            late(bufs[m], xs[m])
            out.append(fp4.linear(bufs[m], w))
            late(bufs[m], xs[m])
            q = fp4.quantize(bufs[m], "nvfp4")
            out.append(fp4.matmul(q, w))
            out.append(fp4.dequantize(q))
        late(xb, x), late(lb, logits)
        out.append(fp4.moe(xb, lb, w13, w2, topk))
        return out

    big.mul_(4096 ** -0.5)
    want = []
    for m in xs:
        q = fp4.quantize(xs[m], "nvfp4")
        want += [fp4.linear(xs[m], w), fp4.matmul(q, w), fp4.dequantize(q)]
    want.append(fp4.moe(x, logits, w13, w2, topk))
    torch.cuda.synchronize()
    if captured:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.stream(main):
            run()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=main):
            got = run()
        for _ in range(3):
            [v.zero_() for v in got]
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    else:
        for _ in range(3):
            with torch.cuda.stream(main):
                got = run()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    fp4.check()
