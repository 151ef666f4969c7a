"""Forward-mode derivatives: the kernels have none, so a call on a tensor with a tangent raises instead of dropping it."""

import pytest
import torch
from torch.autograd import forward_ad

from matterformer_amd import _native
from matterformer_amd.gated_mlp import gated_linear
from matterformer_amd.geometry_ops import radius_attention
from matterformer_amd.rotary import RotaryFrequencies, apply_rotary, rotary_frequencies, rotary_heads
from matterformer_amd.trunk import KnnLocalAttention


def test_a_tangent_counts_as_a_gradient():
    plain = torch.ones(3)
    assert not _native.takes_gradient(plain, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        assert not _native.has_tangent(plain, None) and not _native.takes_gradient(plain)
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                assert _native.takes_gradient(None, plain, dual)
        attn = KnnLocalAttention(64, 2)
        assert not _native.has_tangent(*attn.parameters())


def test_positions_and_frequencies_refuse_a_tangent():
    q, f = torch.zeros(1, 1, 4, 8), rotary_frequencies(8)
    with forward_ad.dual_level():
        pos = forward_ad.make_dual(torch.zeros(1, 4), torch.ones(1, 4))
        with pytest.raises(RuntimeError, match="no derivative"):
            apply_rotary(q, None, pos, f)
        table = forward_ad.make_dual(f.table, torch.ones_like(f.table))
        with pytest.raises(RuntimeError, match="no derivative"):
            apply_rotary(q, None, torch.zeros(1, 4), RotaryFrequencies(table))


def test_cpu_formulations_carry_tangents():
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(2, 4), torch.ones(2, 4))
        assert forward_ad.unpack_dual(gated_linear(x, torch.ones(6, 4))).tangent is not None


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_kernels_refuse_a_tangent(cuda, grad):
    f = rotary_frequencies(8).to(cuda)
    pos = torch.zeros(1, 4, device=cuda)
    bits = torch.full((1, 4, 1), 15, dtype=torch.int32, device=cuda)
    w = torch.ones(6, 8, device=cuda)
    q = torch.ones(1, 1, 4, 32, device=cuda, dtype=torch.bfloat16)

    def dual(*shape, dtype=torch.float32):
        return forward_ad.make_dual(torch.ones(*shape, device=cuda, dtype=dtype), torch.ones(*shape, device=cuda, dtype=dtype))

    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for call in (lambda: gated_linear(dual(2, 8), w), lambda: gated_linear(torch.ones(2, 8, device=cuda), dual(6, 8)),
                     lambda: apply_rotary(dual(1, 1, 4, 8), None, pos, f),
                     lambda: rotary_heads(dual(1, 4, 24), pos, f, heads=1),
                     lambda: radius_attention(q, q, dual(1, 1, 4, 32, dtype=torch.bfloat16), bits)):
            with pytest.raises(NotImplementedError):
                call()
        attn = KnnLocalAttention(64, 2).to(cuda, torch.bfloat16)
        h = dual(1, 4, 64, dtype=torch.bfloat16)
        with torch.no_grad():
            assert attn._use_hip(torch.ones(1, 4, 64, device=cuda, dtype=torch.bfloat16)) and not attn._use_hip(h)
        attn.impl = "triton"
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            attn._use_hip(h)
