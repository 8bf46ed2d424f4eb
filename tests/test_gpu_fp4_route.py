"""GPU: the choice of experts (ops/fp4.py::moe) where scores lie close together."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from ferrite_b200.ops import fp4  # noqa: E402
import test_gpu_fp4_moe as plain  # noqa: E402
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


@pytest.mark.parametrize("with_bias", [False, True])
def test_weights_of_vanishing_scores_still_sum_to_one(with_bias, monkeypatch):
    """Sigmoid scores of 1e-18 to 1e-38: divided by their sum they weigh as much as any others.  All zero in f32: the row is zero."""
    E, D, I, topk = 24, 256, 64, 4
    w13, w2 = experts(E, D, I, 23)
    g = torch.Generator().manual_seed(24)
    low = torch.tensor([0.0, -42.0, -50.0, -60.0, -84.0, -200.0])
    logits = plain.spread_logits(6, E, 25) + low[:, None]
    x = torch.randn(6, D, generator=g)
    bias = torch.zeros(E) if with_bias else None

    def route(logits, bias, topk, score, norm, scale):
        p = torch.sigmoid(logits.double())
        idx = torch.sort(p, dim=-1, descending=True, stable=True).indices[:, :topk]
        w = p.gather(1, idx)
        return idx, w / w.sum(-1, keepdim=True) * scale

    monkeypatch.setattr(plain, "ref_route", route)
    got = fp4.moe(x.cuda(), logits.cuda(), w13, w2, topk, bias=bias.cuda() if with_bias else None, score="sigmoid", scale=1.5)
    check_close(got[:5], *ref_moe(x[:5], logits[:5], w13, w2, topk, score="sigmoid", scale=1.5), torch.float32)
    assert (got[5] == 0).all()
    fp4.check()
