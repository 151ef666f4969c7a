"""Sizes past what the kernels' 32-bit counts hold are refused by the entry points, not cut off (zero-stride views here:
nothing of that size is allocated)."""

import pytest
import torch

from matterformer_amd import gated_mlp, rotary
from matterformer_amd.geometry_ops import radius_attention, radius_tables

FAR = 2 ** 32 + 5  # 5 in 32 bits


@pytest.mark.parametrize("tokens,channels,hidden", [(FAR, 8, 3), (2 ** 30 + 1, 8, 3), (2, FAR, 1), (2, 8, FAR)])
def test_gated_linear(tokens, channels, hidden):
    x = torch.zeros(1, 1).expand(tokens, channels)
    weight = torch.zeros(1, 1).expand(2 * hidden, channels)
    with pytest.raises(RuntimeError, match="gated_linear supports"):
        gated_mlp._arguments(x, weight, None, "silu", None)


@pytest.mark.parametrize("batch,tokens,heads", [(FAR, 1, 1), (1, FAR, 1), (2 ** 16, 2 ** 15, 1), (1, 4, FAR), (1, 4, 2 ** 21)])
def test_rotary(batch, tokens, heads):
    f = rotary.rotary_frequencies(8)
    plan = rotary._Plan(torch.zeros(1, 1, 1).expand(batch, tokens, 1), f.table, 1, 1.0, False)
    zeros = (0,) * 9
    with pytest.raises(RuntimeError, match="rotary positions support"):
        rotary._launch(plan, (0, None, None), zeros, (0, None, None), zeros, (heads, 0, 0), batch=batch, tokens=tokens,
                       head_dim=8, inverse=False, slot_side=0, src_dtype=torch.float32, dst_dtype=torch.float32,
                       device=torch.device("cpu"))


def test_radius_attention():
    bits = torch.zeros(1, 1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="radius_tables supports"):
        radius_tables(bits.expand(FAR, 1, 1))
    for B, H in ((FAR, 1), (1, FAR), (2 ** 16, 2 ** 15)):
        q = torch.zeros(1, 1, 1, 1, dtype=torch.bfloat16).expand(B, H, 1, 32)
        with pytest.raises(RuntimeError, match="radius_attention supports"):
            radius_attention(q, q, q, bits.expand(B, 1, 1))
