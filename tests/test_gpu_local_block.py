"""The rotary local block with a gated MLP as it is used: trunks of local and simplicial blocks, padded and packed, in
inference and training, against the same trunk in float64 on the CPU.

Bars: every operation of a block rounds to bf16, off by at most 2^-8 and by 2^-8 / sqrt(3) in the mean square; about 15
roundings lie between a block's input and its output, so two blocks leave sqrt(30) 2^-8 / sqrt(3) = 1.2e-2 of the norm
(bar 2e-2, that of the trunk's other bf16 tests), and a gradient passes as many again: sqrt(60) 2^-8 / sqrt(3) = 1.7e-2,
times three for sums that cancel (a bias's over tokens): 5e-2."""

import copy

import pytest
import torch

from matterformer_amd.rotary import rotary_frequencies
from matterformer_amd.token_packing import TokenPacking
from matterformer_amd.trunk import AlternatingTrunk

pytestmark = pytest.mark.gpu


def build(schedule, *, d=128, heads=2, gate="silu", layout="half", axes_dim=60, seed=0, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    trunk = AlternatingTrunk(d, heads, len(schedule), knn_k=8, schedule=schedule, mlp_gate=gate, mlp_ratio=2.0,
                             local_rotary=rotary_frequencies(axes_dim, axes=3, base=30.0), local_rotary_layout=layout,
                             local_hip_backward=True, simplicial_precision="bf16_tc")
    for block in trunk.blocks:
        torch.nn.init.normal_(block.ada_ln[-1].weight, std=0.05)
        torch.nn.init.normal_(block.ada_ln[-1].bias, std=0.3)
    return trunk.to(dtype)


def inputs(B=3, N=40, d=128, seed=1):
    gen = torch.Generator().manual_seed(seed)
    counts = torch.tensor([N, 7, 23][:B])
    pad = torch.arange(N)[None] >= counts[:, None]
    x = torch.randn(B, N, d, generator=gen).to(torch.bfloat16)
    cond = torch.randn(B, d, generator=gen).to(torch.bfloat16)
    coords = torch.randn(B, N, 3, generator=gen) * 1.4
    weight = torch.randn(B, N, d, generator=gen).to(torch.bfloat16)
    return x, cond, coords, pad, weight


def reference(trunk, x, cond, coords, pad, weight):
    ref = copy.deepcopy(trunk).cpu().double()
    leaf = x.double().requires_grad_(True)
    out = ref(leaf, cond.double(), coords, pad)
    (out * weight.double()).sum().backward()
    return out.detach(), leaf.grad, {n: p.grad for n, p in ref.named_parameters()}


def rel(got, want):
    return float((got.detach().cpu().double() - want).norm() / want.norm())


@pytest.mark.parametrize("schedule,layout,gate", [(["knn_local", "knn_local"], "half", "silu"),
                                                  (["simplicial", "knn_local"], "interleaved", "gelu_tanh")])
@pytest.mark.parametrize("packed", [False, True])
def test_forward_and_training(cuda, schedule, layout, gate, packed):
    trunk = build(schedule, layout=layout, gate=gate)
    x, cond, coords, pad, weight = inputs()
    want, want_dx, want_grads = reference(trunk, x, cond, coords, pad, weight)
    trunk = trunk.to(cuda)
    trunk.pack_tokens = packed
    args = [t.to(cuda) for t in (cond, coords, pad)]
    with torch.no_grad():
        assert trunk.packable(x.to(cuda)) == packed
        out = trunk(x.to(cuda), *args)
    assert rel(out, want) <= 2e-2
    assert torch.equal(out[pad.to(cuda)], torch.zeros_like(out[pad.to(cuda)]))
    leaf = x.to(cuda).requires_grad_(True)
    out = trunk(leaf, *args)
    (out.float() * weight.to(cuda).float()).sum().backward()
    torch.cuda.synchronize()
    assert all(b.attn._last_impl_used == "triton" for b in trunk.blocks)
    assert rel(out, want) <= 2e-2
    assert rel(leaf.grad, want_dx) <= 5e-2
    for name, param in trunk.named_parameters():
        if want_grads[name] is None:
            continue
        # a key bias shifts a row's logits alike: its gradient is zero but for rounding
        if name.endswith("in_proj_bias") or name.endswith("in_proj.bias"):
            scale = want_grads[name].norm()
            assert float((param.grad.cpu().double() - want_grads[name]).norm()) <= 5e-2 * float(scale), name
            continue
        assert rel(param.grad, want_grads[name]) <= 5e-2, name


def test_packed_equals_padded(cuda):
    """The same rows through both layouts: attention cores see the same operands, so only the summation of the linears
    differs, and with it the bf16 roundings."""
    trunk = build(["knn_local", "knn_local"]).to(cuda)
    x, cond, coords, pad, _ = (t.to(cuda) for t in inputs())
    with torch.no_grad():
        packed = trunk(x, cond, coords, pad)
        trunk.pack_tokens = False
        padded = trunk(x, cond, coords, pad)
    assert rel(packed, padded.cpu().double()) <= 2e-2


def test_float32_training_takes_the_torch_path(cuda):
    trunk = build(["knn_local", "knn_local"], dtype=torch.float32)
    x, cond, coords, pad, weight = inputs()
    want, want_dx, want_grads = reference(trunk, x, cond, coords, pad, weight)
    trunk = trunk.to(cuda)
    leaf = x.to(cuda).float().requires_grad_(True)
    out = trunk(leaf, cond.to(cuda).float(), coords.to(cuda), pad.to(cuda))
    (out * weight.to(cuda).float()).sum().backward()
    assert all(b.attn._last_impl_used == "torch" for b in trunk.blocks)
    # fp32 sums of at most a few hundred terms over two blocks, forward and back
    assert rel(out, want) <= 1e-4 and rel(leaf.grad, want_dx) <= 1e-4
    for name, param in trunk.named_parameters():
        if want_grads[name] is not None:
            assert rel(param.grad, want_grads[name]) <= 1e-3, name


def test_autocast_training_runs_the_kernels(cuda):
    trunk = build(["knn_local", "knn_local"], dtype=torch.float32)
    x, cond, coords, pad, weight = inputs()
    want, want_dx, _ = reference(trunk, x, cond, coords, pad, weight)
    trunk = trunk.to(cuda)
    leaf = x.to(cuda).float().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = trunk(leaf, cond.to(cuda).float(), coords.to(cuda), pad.to(cuda))
    (out.float() * weight.to(cuda).float()).sum().backward()
    assert all(b.attn._last_impl_used == "triton" for b in trunk.blocks)
    assert rel(out, want) <= 2e-2 and rel(leaf.grad, want_dx) <= 5e-2


def test_coordinates_that_ask_for_a_gradient_are_refused(cuda):
    trunk = build(["knn_local"]).to(cuda)
    x, cond, coords, pad, _ = (t.to(cuda) for t in inputs())
    with pytest.raises(RuntimeError, match="no gradient"):
        trunk(x, cond, coords.requires_grad_(True), pad)


def test_captured_inference(cuda):
    trunk = build(["knn_local", "knn_local"]).to(cuda).eval()
    x, cond, coords, pad, _ = (t.to(cuda) for t in inputs())
    packing = TokenPacking(pad)
    gen = torch.Generator().manual_seed(9)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                trunk(x, cond, coords, pad, packing=packing)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = trunk(x, cond, coords, pad, packing=packing)
        for turn in range(3):
            x.copy_(torch.randn(x.shape, generator=gen).to(torch.bfloat16))
            coords.copy_(torch.randn(coords.shape, generator=gen))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, trunk(x, cond, coords, pad, packing=packing)), f"replay {turn}"


def test_one_mask_in_a_captured_step_and_outside_it(cuda):
    """A mask built beforehand, first used by a captured training step: an eager step on it before any replay is right,
    and so is every replay."""
    from matterformer_amd.trunk import KnnLocalAttention, build_knn_mask

    torch.manual_seed(6)
    attn = KnnLocalAttention(64, 2, hip_backward=True).to(cuda, torch.bfloat16)
    gen = torch.Generator().manual_seed(7)
    h = torch.randn(2, 70, 64, generator=gen).to(cuda, torch.bfloat16).requires_grad_(True)
    go = torch.randn(2, 70, 64, generator=gen).to(cuda, torch.bfloat16)
    coords = torch.randn(2, 70, 3, generator=gen).to(cuda)
    leaves = [h, *attn.parameters()]

    def step(mask):
        return torch.autograd.grad(attn(h, mask), leaves, go)

    want = step(build_knn_mask(coords, 8, None, use_hip=True))
    for with_tables in (False, True):
        mask = build_knn_mask(coords, 8, None, use_hip=True, with_tables=with_tables)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(mask)
        assert all(torch.equal(a, b) for a, b in zip(step(mask), want))
        for turn in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want)), turn
            assert all(torch.equal(a, b) for a, b in zip(step(mask), want)), turn


@pytest.mark.parametrize("packed", [False, True])
def test_a_training_trunk_makes_its_tables_once(cuda, packed, monkeypatch):
    from matterformer_amd import geometry_ops

    made, real = [], geometry_ops.radius_tables
    monkeypatch.setattr(geometry_ops, "radius_tables", lambda *a: made.append(a) or real(*a))
    trunk = build(["knn_local", "knn_local", "knn_local"]).to(cuda)
    trunk.pack_tokens = packed
    x, cond, coords, pad, _ = (t.to(cuda) for t in inputs())
    trunk(x, cond, coords, pad).float().sum().backward()
    assert len(made) == 1
    with torch.no_grad():
        trunk(x, cond, coords, pad)
    assert len(made) == 1


@pytest.mark.parametrize("packed", [False, True])
def test_float32_heads_round_once(cuda, packed, monkeypatch):
    """fp32 projections in inference: the 16-bit heads are the turned fp32 rows rounded once, padded or packed."""
    import torch.nn.functional as F

    from matterformer_amd.rotary import rotary_frequencies
    from matterformer_amd.trunk import KnnLocalAttention, build_knn_mask
    from rotary_reference import assert_turned, rotate64

    torch.manual_seed(8)
    f = rotary_frequencies(60, axes=3, base=30.0)
    attn = KnnLocalAttention(128, 2, rotary=f).to(cuda).eval()
    gen = torch.Generator().manual_seed(9)
    h, coords = torch.randn(1, 40, 128, generator=gen).to(cuda), torch.randn(1, 40, 3, generator=gen).to(cuda)
    seen = []
    real = attn._attend
    monkeypatch.setattr(attn, "_attend", lambda q, k, v, mask: seen.extend((q, k, v)) or real(q, k, v, mask))
    with torch.no_grad():
        mask = build_knn_mask(coords, 8, None, use_hip=True)
        if packed:
            hp = h.view(40, 128)
            rows = F.linear(hp, attn.attn.in_proj_weight, attn.attn.in_proj_bias).view(1, 40, 384)
            attn.forward_packed(hp, mask, TokenPacking(torch.zeros(1, 40, dtype=torch.bool, device=cuda)))
        else:
            rows = F.linear(h, attn.attn.in_proj_weight, attn.attn.in_proj_bias)
            attn(h, mask)
    heads = [t.view(1, 40, 2, 64).transpose(1, 2) for t in rows.split(128, dim=-1)]
    assert all(t.dtype == torch.bfloat16 for t in seen) and attn._last_impl_used == "triton"
    for got, part, name in zip(seen[:2], heads[:2], "qk"):
        assert_turned(got, *rotate64(part, coords, f.table, 3, 1.0, "half"), name)
    assert torch.equal(seen[2], heads[2].bfloat16())


def test_float64_modules_in_inference(cuda):
    """The core runs in 16 bits, as it does without rotary positions."""
    from matterformer_amd.trunk import KnnLocalAttention, build_knn_mask

    torch.manual_seed(10)
    attn = KnnLocalAttention(128, 2, rotary=rotary_frequencies(60, axes=3, base=30.0)).to(cuda).double().eval()
    h, coords = torch.randn(1, 40, 128, device=cuda).double(), torch.randn(1, 40, 3, device=cuda)
    with torch.no_grad():
        mask = build_knn_mask(coords, 8, None, use_hip=True)
        out = attn(h, mask)
        assert attn._last_impl_used == "triton"
        attn.impl = "torch"
        want = attn(h, mask)
    assert out.dtype == torch.float64
    # heads, P and the core's output round to bf16 (three roundings of 2^-8 / sqrt(3) in the mean square): 4e-3 of the norm
    assert rel(out, want.cpu()) <= 1e-2


def test_training_after_inference_mode(cuda):
    """A first forward under inference_mode leaves nothing that a gradient cannot be taken through."""
    trunk = build(["knn_local", "knn_local"]).to(cuda)
    x, cond, coords, pad, weight = (t.to(cuda) for t in inputs())
    with torch.inference_mode():
        first = trunk(x, cond, coords, pad)
    leaf = x.clone().requires_grad_(True)
    out = trunk(leaf, cond, coords, pad)
    (out.float() * weight.float()).sum().backward()
    assert leaf.grad is not None and rel(out, first.cpu().double()) <= 2e-2
