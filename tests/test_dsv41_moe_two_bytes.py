"""CPU: what the two-kernel expert layer keeps beside the experts is counted before a model is loaded."""
import pytest
import torch

from ferrite_b200.models.dsv41_config import Dsv41Config
from ferrite_b200.models.dsv41_weights import estimate_device_bytes, moe_two_bytes, padded_inter
from ferrite_b200.ops import fp4
from ferrite_b200.utils.switches import Switches, set_switches


@pytest.mark.parametrize("world", [1, 4, 8])
def test_bytes_of_one_expert_are_those_of_its_tensors(world):
    cfg = Dsv41Config()
    d, Il = cfg.dim, padded_inter(cfg, world) if world > 1 else cfg.moe_inter_dim
    s13, s2 = torch.zeros(2, Il, d // 32, dtype=torch.uint8), torch.zeros(d, Il // 32, dtype=torch.uint8)
    w2 = torch.zeros(d, Il // 2, dtype=torch.uint8)
    padded = torch.nn.functional.pad(w2, (0, (-Il // 2) % 64))
    fp4.Fp4Tensor(padded, fp4.pack_scales(s2), "mxfp4", (d, Il))          # the layout that the layer takes
    extra = fp4.pack_scales(s13).numel() + fp4.pack_scales(s2).numel() + (padded.numel() if padded.numel() > w2.numel() else 0)
    experts = sum(cfg.moe_shape(l)[0] for l in range(cfg.n_layers + cfg.n_mtp_layers))
    assert moe_two_bytes(cfg, world) == extra * experts


def test_the_estimate_follows_the_switch():
    cfg = Dsv41Config()
    base = estimate_device_bytes(cfg, 4)
    try:
        set_switches(Switches(d4_moe_two=True))
        assert estimate_device_bytes(cfg, 4) == base + moe_two_bytes(cfg, 4)
        assert estimate_device_bytes(cfg, 4, moe_two=False) == base
    finally:
        set_switches(None)
    assert estimate_device_bytes(cfg, 4) == base and moe_two_bytes(cfg, 4) > 25e9   # 320 of 608 bytes a row of every down matrix
