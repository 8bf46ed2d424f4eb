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
