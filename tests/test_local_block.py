"""The rotary local block with a gated MLP on the CPU: construction, refusals, the torch path's mathematics."""

import pytest
import torch

from matterformer_amd.rotary import rotary_frequencies
from matterformer_amd.trunk import AdaLNBlock, AlternatingTrunk, KnnLocalAttention, KnnLocalMask, Mlp, build_knn_mask


def test_gated_mlp_module():
    torch.manual_seed(0)
    mlp = Mlp(8, mlp_ratio=2.0, gate="silu").double()
    assert mlp.fc1.weight.shape == (32, 8) and mlp.fc2.weight.shape == (8, 16)
    x = torch.randn(3, 5, 8, dtype=torch.float64)
    gate, up = (x @ mlp.fc1.weight.T + mlp.fc1.bias).chunk(2, dim=-1)
    want = (gate * torch.sigmoid(gate) * up) @ mlp.fc2.weight.T + mlp.fc2.bias
    assert torch.allclose(mlp(x), want, rtol=1e-12, atol=1e-12)
    with pytest.raises(ValueError, match="mlp gate"):
        Mlp(8, gate="tanh")


def test_ungated_mlp_is_unchanged():
    torch.manual_seed(1)
    a = Mlp(8)
    assert list(a.state_dict()) == ["fc1.weight", "fc1.bias", "fc2.weight", "fc2.bias"]
    assert a.fc1.weight.shape == (32, 8) and a.gate is None


def test_autocast_on_the_cpu():
    mlp = Mlp(8, gate="gelu")
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert mlp(torch.randn(4, 8)).dtype == torch.bfloat16


def test_rotary_refusals():
    with pytest.raises(ValueError, match="axes must be 3"):
        KnnLocalAttention(64, 2, rotary=rotary_frequencies(32))
    with pytest.raises(ValueError, match="greater than head_dim"):
        KnnLocalAttention(32, 2, rotary=rotary_frequencies(24, axes=3))
    with pytest.raises(ValueError, match="layout"):
        KnnLocalAttention(64, 2, rotary=rotary_frequencies(24, axes=3), rotary_layout="pairs")
    attn = KnnLocalAttention(64, 2, rotary=rotary_frequencies(24, axes=3))
    mask = KnnLocalMask(torch.zeros(1, 3, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions"):
        attn(torch.zeros(1, 3, 64), mask)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_attention_follows_the_difference_vectors(layout):
    """Moving every atom by one vector changes nothing; without turning (frequencies 0) it is plain local attention."""
    torch.manual_seed(2)
    freqs = rotary_frequencies(24, axes=3, base=20.0)
    attn = KnnLocalAttention(64, 2, rotary=freqs, rotary_layout=layout).double()
    h = torch.randn(2, 9, 64, dtype=torch.float64)
    coords = torch.randn(2, 9, 3)
    pad = torch.zeros(2, 9, dtype=torch.bool)
    pad[1, 6:] = True
    mask = build_knn_mask(coords, 4, pad, use_hip=False)
    moved = KnnLocalMask(mask.idx, allowed=mask.allowed, positions=(coords + torch.tensor([0.5, -1.0, 2.0])))
    out = attn(h, mask, pad)
    assert torch.allclose(out, attn(h, moved, pad), rtol=1e-5, atol=1e-6)
    plain = KnnLocalAttention(64, 2).double()
    plain.load_state_dict(attn.state_dict())
    still = KnnLocalMask(mask.idx, allowed=mask.allowed, positions=torch.zeros_like(coords))
    keep = ~pad
    assert torch.allclose(attn(h, still, pad)[keep], plain(h, mask, pad)[keep], rtol=1e-9, atol=1e-9)


def test_trunk_with_every_option_trains_on_the_cpu():
    torch.manual_seed(3)
    trunk = AlternatingTrunk(64, 2, 2, knn_k=4, mlp_gate="silu", local_rotary=rotary_frequencies(30, axes=3, base=50.0),
                             local_hip_backward=True, simplicial_precision="ieee_fp32").double()
    for block in trunk.blocks:
        torch.nn.init.normal_(block.ada_ln[-1].weight, std=0.05)
    x, cond = torch.randn(2, 7, 64, dtype=torch.float64), torch.randn(2, 64, dtype=torch.float64)
    coords, pad = torch.randn(2, 7, 3), torch.zeros(2, 7, dtype=torch.bool)
    pad[0, 5:] = True
    out = trunk(x, cond, coords, pad)
    out.square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in trunk.parameters())
    assert trunk.blocks[1].attn._last_impl_used == "torch"
    assert isinstance(trunk.blocks[0], AdaLNBlock) and trunk.blocks[0].mlp.gate == "silu"


def test_another_table_of_frequencies_takes_effect():
    """Assigned, or changed in place, after a forward: the next one turns by it (its copy on the device too)."""
    torch.manual_seed(4)
    attn = KnnLocalAttention(64, 2, rotary=rotary_frequencies(24, axes=3, base=20.0)).double()
    h, coords = torch.randn(1, 9, 64, dtype=torch.float64), torch.randn(1, 9, 3) * 3
    mask = build_knn_mask(coords, 4, None, use_hip=False)
    meta = torch.device("meta")  # another device than the table's

    def fresh():
        other = KnnLocalAttention(64, 2, rotary=rotary_frequencies(24, axes=3, base=20.0)).double()
        other.load_state_dict(attn.state_dict())
        other.rotary = attn.rotary
        return other(h, mask)

    first, held = attn(h, mask), attn._rotary(meta)
    assert attn._rotary(meta) is held  # one copy a device, while the table stays
    attn.rotary = rotary_frequencies(24, axes=3, base=500.0)
    second = attn(h, mask)
    assert not torch.allclose(first, second) and torch.equal(second, fresh())
    assert attn._rotary(meta) is not held
    held = attn._rotary(meta)
    attn.rotary.table.mul_(0.5)
    third = attn(h, mask)
    assert not torch.allclose(second, third) and torch.equal(third, fresh())
    assert attn._rotary(meta) is held  # the same copy, changed with it (a captured graph reads it)


@pytest.mark.gpu
def test_another_table_of_frequencies_takes_effect_on_the_gpu(cuda):
    """The module's copy there follows an assignment and a change in place, also one behind a captured graph."""
    torch.manual_seed(5)
    attn = KnnLocalAttention(64, 2, rotary=rotary_frequencies(24, axes=3, base=20.0)).to(cuda, torch.bfloat16)
    h, coords = torch.randn(1, 9, 64).to(cuda, torch.bfloat16), torch.randn(1, 9, 3, device=cuda) * 3
    mask = build_knn_mask(coords, 4, None, use_hip=True)

    def fresh():
        other = KnnLocalAttention(64, 2, rotary=attn.rotary).to(cuda, torch.bfloat16)
        other.load_state_dict(attn.state_dict())
        return other(h, mask)

    with torch.no_grad():
        first = attn(h, mask)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attn(h, mask)
        attn.rotary.table.mul_(2.0)
        second = attn(h, mask)
        graph.replay()
        torch.cuda.synchronize()
        assert not torch.equal(first, second) and torch.equal(second, fresh()) and torch.equal(out, second)
        attn.rotary = rotary_frequencies(24, axes=3, base=500.0)
        third = attn(h, mask)
        assert not torch.equal(second, third) and torch.equal(third, fresh())
        filler = [torch.full((12,), 7.0, dtype=torch.float64, device=cuda) for _ in range(64)]
        graph.replay()  # as it was captured
        torch.cuda.synchronize()
        assert torch.equal(out, second) and len(filler) == 64


def test_tables_are_kept_only_by_a_mask_built_with_them(monkeypatch):
    """A mask keeps no tables of a call on it (which may have been captured, or on another stream), and drops those it was
    built with when its bits change."""
    from matterformer_amd import geometry_ops

    made = []

    def make(bits, blocks):
        made.append(bits)
        return object()

    monkeypatch.setattr(geometry_ops, "radius_tables", make)
    bits = torch.ones(1, 3, 1, dtype=torch.int32)
    mask = KnnLocalMask(torch.zeros(1, 3, 1, dtype=torch.int32), bits=bits)
    assert mask.tables() is not mask.tables() and len(made) == 2
    mask = KnnLocalMask(mask.idx, bits=bits, with_tables=True)
    assert len(made) == 3 and mask.tables() is mask.tables() and len(made) == 3
    bits.zero_()
    assert mask.tables() is not mask.tables() and len(made) == 5
    mask = KnnLocalMask(mask.idx, bits=bits, with_tables=True)
    mask.bits = torch.ones(1, 3, 1, dtype=torch.int32)
    assert mask.tables() is not mask.tables() and made[-1] is mask.bits
