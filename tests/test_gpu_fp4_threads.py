"""GPU: 4-bit operators of two host threads that share one stream, so that launches of different calls mix."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

from ferrite_b200.ops import fp4, mx  # noqa: E402
from ferrite_b200.ops import quant as Q  # noqa: E402


def grouped_product(g):
    """A call of the expert-grouped tcgen05 product, which lets its dependents start before it takes tensor memory."""
    E, N, K, counts, bn = 2, 256, 512, [40, 24], 64
    packed, scales = zip(*[Q.quant_fp4_weight(torch.randn(N, K, generator=g) * 0.05) for _ in range(E)])
    packed, sfa = torch.stack(packed).cuda(), mx.pack_weight_scales(torch.stack(scales).cuda())
    xq, xs = Q.fp8_act_quant(torch.randn(sum(counts), K, generator=g))
    xq, xs = xq.to(torch.float8_e4m3fn).cuda(), xs.cuda()
    tiles, n_tiles, _ = mx.make_tiles(torch.tensor(counts, dtype=torch.int32, device="cuda"), bn)
    status = torch.zeros(4, dtype=torch.int32, device="cuda")

    def call():
        out = torch.zeros(sum(counts), N, device="cuda")
        mx.mx_gemm_grouped(packed, sfa, xq, xs, tiles, n_tiles, out, bn, status)
        return out
    return call


def test_two_threads_on_one_stream():
    """Calls of two kernels each (linear of several rows, linear of many, the expert layer) on one stream, with another tcgen05
    product between their launches wherever the threads happen to meet."""
    g = torch.Generator().manual_seed(3)
    T, E, D, I, topk = 4, 8, 512, 128, 2
    w = fp4.quantize(torch.randn(640, D, generator=g).cuda(), "nvfp4")
    w13, w2 = fp4.quantize(torch.randn(E, 2, I, D, generator=g).cuda()), fp4.quantize(torch.randn(E, D, I, generator=g).cuda())
    logits = torch.randn(T, E, generator=g).cuda()
    x, few, many = (torch.randn(n, D, generator=g).cuda() for n in (T, 24, 300))
    product = grouped_product(g)
    jobs = [[lambda: fp4.moe(x, logits, w13, w2, topk), lambda: fp4.linear(few, w), lambda: fp4.linear(many, w)],
            [product, lambda: fp4.linear(few, w), lambda: fp4.moe(x, logits, w13, w2, topk)]]
    want = [[j() for j in js] for js in jobs]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(stream):
            for _ in range(200):
                got[i].append([j() for j in jobs[i]])

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    for i in (0, 1):
        assert len(got[i]) == 200
        for ys in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(ys, want[i]))
    fp4.check()
