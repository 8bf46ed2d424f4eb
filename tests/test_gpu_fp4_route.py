"""GPU: the choice of experts (ops/fp4.py::moe) where scores lie close together."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from ferrite_b200.ops import fp4  # noqa: E402
from test_gpu_fp4_moe import check_close, experts, ref_moe  # noqa: E402


@pytest.mark.parametrize("T", [3, 32])       # scores shared by threads, and a token per warp
@pytest.mark.parametrize("score", ["sigmoid", "sqrtsoftplus", "softmax"])
def test_scores_a_few_units_apart(score, T):
    """Logits near -30, one unit in the last place (2^-19) from the next: the scores, about exp(z) or its root, are 16 or 8 units
    apart.  A score in f32 is off by under 4 units (exponential 2, logarithm 1, sum, quotient and root half of one each, the
    root halving what comes in), so the order of 64 bits is the order that counts."""
    E, D, I, topk = 384, 128, 32, 5
    w13, w2 = experts(E, D, I, 21)
    g = torch.Generator().manual_seed(22)
    steps = torch.stack([torch.randperm(E, generator=g) for _ in range(T)])
    logits = -30.0 + (steps + 7 * torch.arange(T)[:, None]).float() * 2.0 ** -19
    assert all(len(row.unique()) == E for row in logits)
    bias = torch.zeros(E)
    if score == "softmax":       # a largest logit of 0, kept out of the choice by its bias
        logits[:, 100], bias[100] = 0.0, -2.0
    x = torch.randn(T, D, generator=g).cuda()
    got = fp4.moe(x, logits.cuda(), w13, w2, topk, bias=bias.cuda(), score=score)
    check_close(got, *ref_moe(x, logits, w13, w2, topk, bias=bias, score=score), torch.float32)
    fp4.check()
