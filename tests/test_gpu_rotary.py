"""mf_rotary against the definition in float64: types, layouts, parts of the head, axes, strides, packed rows,
positions far out, gradients, streams and captured graphs."""

import pytest
import torch

from matterformer_amd.rotary import RotaryFrequencies, apply_rotary, rotary_frequencies, rotary_heads
from matterformer_amd.token_packing import TokenPacking
from rotary_reference import assert_turned, rotate64

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen).to(dtype)


CASES = [
    # B, H, KV, N, D, R, axes
    (1, 1, 1, 1, 8, 8, 1),
    (2, 3, 1, 5, 32, 24, 3),
    (1, 8, 8, 29, 32, 30, 3),
    (3, 4, 2, 181, 64, 60, 3),
    (2, 12, 3, 67, 128, 128, 1),
    (1, 2, 2, 7, 20, 8, 2),      # head_dim no multiple of 8: one element at a time
    (2, 1, 1, 33, 256, 256, 2),
    (1, 40, 40, 3, 256, 10, 1),  # more chunks a token than a workgroup takes
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,H,KV,N,D,R,axes", CASES)
def test_heads_and_gradients(cuda, dtype, layout, B, H, KV, N, D, R, axes):
    print(f"rotary B={B} H={H} KV={KV} N={N} D={D} R={R} axes={axes} {layout} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(B * 1000 + N + D)
    f = RotaryFrequencies(rotary_frequencies(R, axes=axes, base=100.0).table, axes, 1.25)
    pos = torch.randn(B, N, axes, generator=gen) * 20
    rows = _randn(gen, B, N, (H + 2 * KV) * D, dtype=dtype)
    q, k, v = rows.split((H * D, KV * D, KV * D), dim=-1)
    heads = [t.view(B, N, -1, D).transpose(1, 2) for t in (q, k, v)]
    grads = [_randn(gen, *h.shape, dtype=dtype) for h in heads]
    leaf = rows.to(cuda).requires_grad_(True)
    fd = f.to(cuda)
    out = rotary_heads(leaf, pos.to(cuda), fd, heads=H, kv_heads=KV, layout=layout)
    (drows,) = torch.autograd.grad(out, leaf, [g.to(cuda) for g in grads])
    dq, dk, dv = drows.split((H * D, KV * D, KV * D), dim=-1)
    back = [t.reshape(B, N, -1, D).transpose(1, 2) for t in (dq, dk, dv)]
    for i, name in enumerate("qk"):
        assert out[i].is_contiguous()
        assert_turned(out[i], *rotate64(heads[i], pos, f.table, axes, f.gain, layout), name)
        assert_turned(back[i], *rotate64(grads[i], pos, f.table, axes, f.gain, layout, inverse=True), "d" + name)
    assert torch.equal(out[2].cpu(), heads[2]) and torch.equal(back[2].cpu(), grads[2])
    # the same heads as strided views, each with a gradient of its own
    a, b = (t.view(B, N, -1, D).transpose(1, 2).requires_grad_(True)
            for t in rows.to(cuda).split((H * D, KV * D, KV * D), dim=-1)[:2])
    views = apply_rotary(a, b, pos.to(cuda), fd, layout=layout)
    da, db = torch.autograd.grad(views, (a, b), [g.to(cuda) for g in grads[:2]])
    assert torch.equal(views[0], out[0]) and torch.equal(views[1], out[1])
    assert torch.equal(da, back[0]) and torch.equal(db, back[1])


@pytest.mark.parametrize("ptype", [torch.float32, torch.float64, torch.int32, torch.int64])
def test_far_positions_and_types(cuda, ptype):
    far = 2 ** 24 - 40 if ptype == torch.float32 else 10 ** 7
    pos = (far + torch.arange(33))[None].to(ptype)
    gen = torch.Generator().manual_seed(5)
    x = _randn(gen, 2, 2, 33, 64, dtype=torch.float32)
    f = rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096)
    got, none = apply_rotary(x.to(cuda), None, pos.to(cuda), f.to(cuda))
    assert none is None
    # fp64 angles: 10^7 rounds to 2^-29 rad, far below the bound
    assert_turned(got, *rotate64(x, pos.expand(2, 33), f.table, 1, f.gain, "half"), str(ptype))


def test_unturned_entries_keep_their_values(cuda):
    x = torch.randn(1, 2, 4, 16)
    x[..., 8:] = float("inf")
    x[0, 1, 2, 9] = float("nan")
    f = rotary_frequencies(8)
    got, _ = apply_rotary(x.to(cuda), None, torch.arange(4)[None].to(cuda), f.to(cuda))
    assert torch.equal(got[..., 8:].cpu().nan_to_num(7.0, 9.0), x[..., 8:].nan_to_num(7.0, 9.0))
    assert torch.isfinite(got[..., :8]).all()


@pytest.mark.parametrize("offset,stride", [(1, 64), (8, 65), (0, 70)])
def test_unaligned_views(cuda, offset, stride):
    """Bases and token strides that are no multiple of 16 bytes."""
    gen = torch.Generator().manual_seed(6)
    base = _randn(gen, offset + 11 * stride + 64, dtype=torch.bfloat16).to(cuda)
    x = base.as_strided((1, 2, 11, 32), (0, 32, stride, 1), offset)
    f = rotary_frequencies(20)
    got, _ = apply_rotary(x, None, torch.arange(11, device=cuda)[None], f.to(cuda))
    want = rotate64(x.cpu(), torch.arange(11)[None], f.table, 1, 1.0, "half")
    assert_turned(got, *want, "unaligned")


def test_expanded_inputs_and_gradients(cuda):
    """Broadcast heads (stride 0) as input, the all-ones gradient of a sum as output gradient."""
    gen = torch.Generator().manual_seed(7)
    one = _randn(gen, 1, 1, 9, 16, dtype=torch.float32)
    leaf = one.to(cuda).requires_grad_(True)
    f = rotary_frequencies(16)
    pos = torch.arange(9)[None]
    got, _ = apply_rotary(leaf.expand(2, 4, 9, 16), None, pos.to(cuda), f.to(cuda))
    assert_turned(got, *rotate64(one.expand(2, 4, 9, 16), pos.expand(2, 9), f.table, 1, 1.0, "half"), "expanded")
    got.sum().backward()
    want, bound = rotate64(torch.ones(1, 1, 9, 16), pos, f.table, 1, 1.0, "half", inverse=True)
    # eight shared copies: eight times one gradient, summed in fp32 (7 roundings of at most 8 |g| 2^-24)
    err = (leaf.grad.cpu().double() - 8 * want).abs()
    assert torch.all(err <= 8 * (bound * 7 * 2.0 ** -24 + want.abs() * 2.0 ** -24) + 7 * 8 * 1.5 * 2.0 ** -24)


def test_gradient_against_differences(cuda):
    gen = torch.Generator().manual_seed(8)
    x = _randn(gen, 1, 2, 6, 12, dtype=torch.float32).to(cuda)
    go = _randn(gen, 1, 2, 6, 12, dtype=torch.float32).to(cuda)
    step = _randn(gen, 1, 2, 6, 12, dtype=torch.float32).to(cuda)
    pos = torch.randn(1, 6, 3, generator=gen).to(cuda)
    f = rotary_frequencies(12, axes=3, base=10.0).to(cuda)
    leaf = x.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(apply_rotary(leaf, None, pos, f)[0], leaf, go)
    plus, minus = (apply_rotary(x + s * step, None, pos, f)[0].double() for s in (0.5, -0.5))
    diff = float(((plus - minus) * go.double()).sum())
    slope = float((grad.double() * step.double()).sum())
    # the map is linear; 144 entries, values below 8, each off by at most 10 roundings of 2^-24
    assert abs(diff - slope) <= 144 * 2 * 8 * 8 * 10 * 2.0 ** -24


@pytest.mark.parametrize("src,dst", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                     (torch.float16, torch.float32)])
@pytest.mark.parametrize("D", [32, 20])
def test_packed_rows(cuda, src, dst, D):
    """Packed rows through the slot map: each molecule's valid atoms first, empty slots zero, and the gradient."""
    gen = torch.Generator().manual_seed(9)
    B, N, H = 3, 11, 2
    pad = torch.rand(B, N, generator=gen) < 0.4
    pad[1] = True  # a molecule without an atom
    pad[0] = False
    packing = TokenPacking(pad.to(cuda))
    rows = _randn(gen, packing.tokens, 3 * H * D, dtype=src)
    coords = torch.randn(B, N, 3, generator=gen) * 5
    pos = packing.compact(coords.to(cuda))
    f = rotary_frequencies(18, axes=3, base=30.0)
    leaf = rows.to(cuda).requires_grad_(True)
    out = packing.to_rotary_heads(leaf, H, D, dst, pos, f.to(cuda), "interleaved")
    plain = torch.zeros(3, B, packing.width, H, D, dtype=src)
    plain[:, packing.mol.cpu(), packing.pos.cpu()] = rows.view(-1, 3, H, D).transpose(0, 1)
    plain = plain.permute(0, 1, 3, 2, 4)
    grads = [_randn(gen, B, H, packing.width, D, dtype=dst) for _ in range(3)]
    (drows,) = torch.autograd.grad(out, leaf, [g.to(cuda) for g in grads])
    back = drows.cpu().view(-1, 3, H, D)
    for i in range(3):
        assert out[i].dtype == dst and out[i].shape == (B, H, packing.width, D)
        if i < 2:
            assert_turned(out[i], *rotate64(plain[i], pos, f.table, 3, 1.0, "interleaved"), "packed")
            want, bound = rotate64(grads[i], pos, f.table, 3, 1.0, "interleaved", inverse=True)
        else:
            assert torch.equal(out[i].cpu(), plain[i].to(dst))
            want, bound = grads[i].double(), torch.zeros(grads[i].shape, dtype=torch.float64)
        at = (packing.mol.cpu(), slice(None), packing.pos.cpu())
        assert_turned(back[:, i], want[at], bound[at], "packed gradient")


@pytest.mark.parametrize("B,N", [(0, 5), (2, 0)])
def test_empty(cuda, B, N):
    f = rotary_frequencies(8).to(cuda)
    rows = torch.zeros(B, N, 3 * 8, device=cuda, requires_grad=True)
    out = rotary_heads(rows, torch.zeros(B, N, device=cuda), f, heads=1)
    (g,) = torch.autograd.grad(out, rows, [torch.ones_like(t) for t in out])
    assert out[0].shape == (B, 1, N, 8) and g.shape == rows.shape


def test_gpu_refusals(cuda):
    f = rotary_frequencies(8)
    q = torch.zeros(1, 1, 4, 8, device=cuda)
    with pytest.raises(RuntimeError, match="on the device of the heads"):
        apply_rotary(q, None, torch.zeros(1, 4, device=cuda), f)
    with pytest.raises(RuntimeError, match="on the device of the heads"):
        apply_rotary(q, None, torch.zeros(1, 4), f.to(cuda))
    with pytest.raises(RuntimeError, match="bfloat16, float16 and float32"):
        apply_rotary(q.double(), None, torch.zeros(1, 4, device=cuda), f.to(cuda))
    with pytest.raises(RuntimeError, match="head_dim up to 256"):
        apply_rotary(torch.zeros(1, 1, 4, 264, device=cuda), None, torch.zeros(1, 4, device=cuda), f.to(cuda))


def test_stream_and_graph(cuda):
    """Forward and backward on a side stream, then captured and replayed with eager work in between."""
    gen = torch.Generator().manual_seed(10)
    rows = _randn(gen, 2, 40, 3 * 64, dtype=torch.bfloat16).to(cuda).requires_grad_(True)
    pos = torch.randn(2, 40, 3, generator=gen).to(cuda)
    f = rotary_frequencies(18, axes=3).to(cuda)
    go = [_randn(gen, 2, 2, 40, 32, dtype=torch.bfloat16).to(cuda) for _ in range(3)]

    def once():
        out = rotary_heads(rows, pos, f, heads=2)
        grads = torch.autograd.grad(out, rows, go)
        return [*(t.detach() for t in out), *grads]

    want = [t.clone() for t in once()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for turn in range(3):
        with torch.no_grad():
            rows.copy_(_randn(gen, 2, 40, 3 * 64, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, once())), f"replay {turn}"


def test_positions_changed_before_the_gradient_are_an_error(cuda):
    f = rotary_frequencies(16).to(cuda)
    rows = torch.randn(1, 4, 3 * 16, device=cuda, requires_grad=True)
    pos = torch.arange(4, device=cuda)[None].float()
    out = rotary_heads(rows, pos, f, heads=1)
    pos += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out[0].sum().backward()


def test_two_calls_in_flight_and_long_rows(cuda):
    """Two graphs of one leaf, their gradients in either order; a batch whose elements pass 2^31."""
    f = rotary_frequencies(16).to(cuda)
    rows = torch.randn(2, 5, 3 * 16, device=cuda, requires_grad=True)
    a = rotary_heads(rows, torch.arange(5, device=cuda)[None], f, heads=1)
    b = rotary_heads(rows, torch.arange(5, device=cuda)[None] + 7, f, heads=1)
    one = [torch.ones_like(t) for t in a]
    (gb,) = torch.autograd.grad(b, rows, one)
    (ga,) = torch.autograd.grad(a, rows, one)
    again = rotary_heads(rows, torch.arange(5, device=cuda)[None], f, heads=1)
    assert torch.equal(torch.autograd.grad(again, rows, one)[0], ga) and not torch.equal(ga, gb)
    big = torch.zeros(2, 700000, 3 * 2 * 256, dtype=torch.bfloat16, device=cuda)  # 2.15e9 elements
    big[1, -1] = 1.0
    f = rotary_frequencies(256).to(cuda)
    pos = torch.zeros(1, 700000, dtype=torch.int32, device=cuda)
    q, k, v = rotary_heads(big, pos, f, heads=2)
    for t in (q, k, v):
        assert torch.equal(t[1, :, -1], torch.ones(2, 256, dtype=torch.bfloat16, device=cuda))
        assert float(t[0, :, -1].abs().max()) == 0.0 and float(t[1, :, -2].abs().max()) == 0.0


@pytest.mark.parametrize("H,KV", [(0, 2), (2, 0), (0, 0)])
def test_no_heads(cuda, H, KV):
    f = rotary_frequencies(8).to(cuda)
    q, k = (torch.ones(2, h, 5, 8, device=cuda, requires_grad=True) for h in (H, KV))
    pos = torch.zeros(2, 5, device=cuda)
    out = apply_rotary(q, k, pos, f)
    grads = torch.autograd.grad(out, (q, k), [torch.ones_like(t) for t in out])
    for t, o, g in zip((q, k), out, grads):
        assert torch.equal(o, t.detach()) and torch.equal(g, t.detach())
