"""Gradients of radius_attention (mf_radius_attn_bwd) against float64, element by element.

Tolerances, from the arithmetic: u = 2^-24, t = eps / 2 of the operands' type.
  logits     |S' - S| <= es_i = (D + 4) u scale max_j sum|q_i k_j|
  lse        the forward sums P rounded to the type: |lse' - lse| <= es_i + t + N u
  P          relative ep_i = 2 es_i + t + N u + 2^-20 (hardware exp2 of an argument below 2^4)
  out        |out' - out| <= (ep_i + t + N u) sum_j P|v| + t |out|
  dP         |dP' - dP| <= (D + 1) u sum|go v|;  delta alike with out' for out, and grad_lse once rounded (u)
  dS         |dS' - dS| <= P (ep (|dP| + |delta|) + errors of dP and delta), then rounded: t |dS|; fp16 keeps
             dS 2^e with 2^e 2 max|go| max|v| in [2^13, 2^14): a step below the normal numbers is
             2^-25 2^-e <= 2^-38 (2 max|go| max|v| + max|dlse|)
  dv         (ep + t + (N + 1) u) sum_i P|go|, fp16: + 2^-25 sum_i |go| for P below the normal numbers
  dq, dk     scale times the sums of dS's error and (N + 2) u |dS| against |k| or |q|
and one rounding of each output, t relative or half the smallest subnormal.  Products of two of these errors are left
out; each relative one is below 2^-5 here, so the sum is taken 1 + 2^-4 times."""

import math

import pytest
import torch

from matterformer_amd.geometry_ops import radius_attention, radius_tables

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def pack(allowed):
    B, N, _ = allowed.shape
    W = (N + 31) // 32
    full = torch.zeros(B, N, W * 32, dtype=torch.int64)
    full[..., :N] = allowed
    word = (full.view(B, N, W, 32) << torch.arange(32)).sum(-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def blocks(allowed):
    B, N, _ = allowed.shape
    NB = (N + 63) // 64
    full = torch.zeros(B, NB * 64, NB * 64, dtype=torch.bool)
    full[:, :N, :N] = allowed
    return full.view(B, NB, 64, NB, 64).any(4).any(2).to(torch.uint8)


def mask_of(kind, B, N, gen):
    eye = torch.eye(N, dtype=torch.bool)[None].expand(B, N, N)
    if kind == "dense":
        return torch.ones(B, N, N, dtype=torch.bool)
    if kind == "self":
        return eye.clone()
    if kind == "none":
        return torch.zeros(B, N, N, dtype=torch.bool)
    if kind == "band":  # most 64 x 64 tiles are empty
        d = (torch.arange(N)[:, None] - torch.arange(N)[None]).abs()
        return (d <= 20)[None].expand(B, N, N).clone()
    allowed = (torch.rand(B, N, N, generator=gen) < 0.15) | eye
    if kind == "ragged":  # padding behind, one molecule without an atom, rows and columns without a partner
        counts = torch.randint(1, N + 1, (B,), generator=gen)
        counts[0] = 0
        valid = torch.arange(N)[None] < counts[:, None]
        allowed &= valid[:, :, None] & valid[:, None]
        allowed[-1, N // 3] = False
        allowed[-1, :, N // 2] = False
    return allowed


def reference(q, k, v, go, allowed, scale, glse=None):
    """(out, lse, dq, dk, dv) in float64, and the bounds of the gradients before the last rounding."""
    dtype, N, D = q.dtype, q.shape[-2], q.shape[-1]
    t = torch.finfo(dtype).eps / 2
    Q, K, V, G = (x.double() for x in (q, k, v, go))
    A = allowed.to(q.device)[:, None]
    s = scale * (Q @ K.mT)
    top = s.masked_fill(~A, -math.inf).amax(-1, keepdim=True)
    has = torch.isfinite(top)
    e = torch.where(A, torch.exp(s - torch.where(has, top, 0.0)), 0.0)
    total = e.sum(-1, keepdim=True)
    P = e / torch.where(has, total, 1.0)
    lse = torch.where(has, torch.where(has, top, 0.0) + torch.log(torch.where(has, total, 1.0)), 0.0)[..., 0]
    out = P @ V
    dP = G @ V.mT
    delta = (G * out).sum(-1, keepdim=True)
    gl = torch.zeros_like(lse) if glse is None else glse.double()
    delta = delta - gl[..., None]
    dS = P * (dP - delta)
    es = (D + 4) * U * abs(scale) * torch.where(A, Q.abs() @ K.abs().mT, 0.0).amax(-1, keepdim=True)
    ep = 2 * es + t + N * U + 2.0 ** -20
    eo = (ep + t + N * U) * (P @ V.abs()) + t * out.abs()
    edp = (D + 1) * U * (G.abs() @ V.abs().mT)
    edelta = (G.abs() * eo).sum(-1, keepdim=True) + (D + 1) * U * (G * out).abs().sum(-1, keepdim=True) + U * gl.abs()[..., None]
    eds = P * (ep * (dP.abs() + delta.abs()) + edp + edelta)
    flush = 0.0
    ev = (ep + t + (N + 1) * U) * P
    if dtype == torch.float16:
        peak = 2 * G.norm(dim=-1).amax(-1) * V.norm(dim=-1).amax(-1) + gl.abs().amax(-1)
        flush = torch.where(A, 2.0 ** -38 * peak[..., None, None], 0.0)
        ev = ev + torch.where(A, 2.0 ** -25, 0.0)
    mds = dS.abs() + eds
    eds = eds + t * mds + flush + (N + 2) * U * mds
    sc = abs(scale)
    bounds = (sc * (eds @ K.abs()), sc * (eds.mT @ Q.abs()), ev.mT @ G.abs())
    grads = (scale * (dS @ K), scale * (dS.mT @ Q), P.mT @ G)
    return out, lse, grads, [b * (1 + 2.0 ** -4) for b in bounds]


def check(got, want, bound, what):
    fi = torch.finfo(got.dtype)
    tol = bound + (want.abs() + bound) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    err = (got.double() - want).abs()
    over = err - tol
    assert torch.all(over <= 0), f"{what}: off by {float(err.max()):.3e}, {float(over.max()):.3e} past the bound"


def operands(B, H, N, D, dtype, seed, device, std=1.0, gstd=0.1):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = ((torch.randn(B, H, N, D, generator=gen) * std).to(dtype).to(device) for _ in range(3))
    go = (torch.randn(B, H, N, D, generator=gen) * gstd).to(dtype).to(device)
    return q, k, v, go, gen


def gradients(q, k, v, go, bits, bm, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = radius_attention(*leaves, bits, bm, **kw)
    return torch.autograd.grad(out, leaves, go)


CASES = [
    # B, H, N, D, mask
    (1, 1, 1, 32, "dense"), (2, 3, 5, 64, "dense"), (3, 2, 29, 32, "ragged"), (1, 2, 63, 128, "random"),
    (2, 1, 64, 64, "random"), (1, 2, 65, 32, "dense"), (2, 2, 100, 64, "ragged"), (1, 1, 129, 128, "ragged"),
    (1, 2, 300, 64, "band"), (2, 1, 181, 64, "ragged"), (1, 1, 257, 32, "self"), (1, 1, 70, 128, "none"),
    (1, 1, 200, 128, "dense"), (1, 1, 4500, 32, "band"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,N,D,kind", CASES)
def test_gradients(cuda, dtype, B, H, N, D, kind):
    print(f"radius gradient B={B} H={H} N={N} D={D} {kind} {dtype}", flush=True)
    q, k, v, go, gen = operands(B, H, N, D, dtype, N * 10 + D, cuda)
    allowed = mask_of(kind, B, N, gen)
    bits, bm = pack(allowed).to(cuda), blocks(allowed).to(cuda)
    got = gradients(q, k, v, go, bits, bm)
    _, _, want, bounds = reference(q, k, v, go, allowed, D ** -0.5)
    for g, w, b, name in zip(got, want, bounds, ("dq", "dk", "dv")):
        check(g, w, b, name)
    again = gradients(q, k, v, go, bits, None)  # without the block mask, and a second call: the same bits
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale,std,gstd", [(-0.3, 1.0, 0.1), (0.125, 4.0, 1e-4), (0.125, 0.05, 50.0), (0.0, 1.0, 0.1)])
def test_scales_and_magnitudes(cuda, dtype, scale, std, gstd):
    """Negative and zero scale, sharp and flat rows, gradients near fp16's smallest and largest numbers."""
    q, k, v, go, gen = operands(2, 2, 90, 64, dtype, 5, cuda, std, gstd)
    allowed = mask_of("ragged", 2, 90, gen)
    got = gradients(q, k, v, go, pack(allowed).to(cuda), None, scale=scale)
    _, _, want, bounds = reference(q, k, v, go, allowed, scale)
    for g, w, b, name in zip(got, want, bounds, ("dq", "dk", "dv")):
        check(g, w, b, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_through_lse(cuda, dtype):
    q, k, v, go, gen = operands(2, 2, 77, 32, dtype, 6, cuda)
    allowed = mask_of("ragged", 2, 77, gen)
    bits = pack(allowed).to(cuda)
    glse = torch.randn(2, 2, 77, generator=gen).to(cuda)
    _, ref_lse, want, bounds = reference(q, k, v, go, allowed, 32 ** -0.5, glse)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, lse, out32 = radius_attention(*leaves, bits, return_lse=True, return_fp32=True)
    assert not out32.requires_grad
    assert float((lse.detach().double() - ref_lse).abs().max()) < 0.02
    for g, w, b, name in zip(torch.autograd.grad((out, lse), leaves, (go, glse)), want, bounds, ("dq", "dk", "dv")):
        check(g, w, b, name)
    # lse alone: no gradient of v, and out's gradient taken as zero
    _, _, want, bounds = reference(q, k, v, torch.zeros_like(go), allowed, 32 ** -0.5, glse)
    out, lse = radius_attention(*leaves, bits, return_lse=True)
    grads = torch.autograd.grad(lse, leaves, glse)
    for g, w, b, name in zip(grads, want, bounds, ("dq", "dk", "dv")):
        check(g, w, b, name)
    assert torch.equal(grads[2], torch.zeros_like(v))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_without_a_partner_reach_nothing(cuda, dtype, bad):
    q, k, v, go, gen = operands(2, 2, 100, 64, dtype, 7, cuda)
    allowed = mask_of("ragged", 2, 100, gen)
    bits = pack(allowed).to(cuda)
    want = gradients(q, k, v, go, bits, None)
    no_key = ~allowed.any(2)  # queries without a key
    no_query = ~allowed.any(1)
    leaves = [t.clone() for t in (q, k, v)]
    leaves[0].masked_fill_(no_key.to(cuda)[:, None, :, None], bad)
    leaves[1].masked_fill_(no_query.to(cuda)[:, None, :, None], bad)
    grad = go.masked_fill(no_key.to(cuda)[:, None, :, None], bad)
    got = gradients(*leaves, grad, bits, None)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_layouts(cuda):
    """Operands and gradient as transposed views and at an odd element offset; an expanded gradient."""
    B, H, N, D = 2, 2, 70, 32
    q, k, v, go, gen = operands(B, H, N, D, torch.bfloat16, 8, cuda)
    allowed = mask_of("random", B, N, gen)
    bits = pack(allowed).to(cuda)
    want = gradients(q, k, v, go, bits, None)
    rows = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, go)]
    assert all(torch.equal(a, b) for a, b in zip(gradients(*rows, bits, None), want))
    odd = torch.empty(go.numel() + 1, dtype=go.dtype, device=cuda)[1:].view(go.shape).copy_(go)
    assert odd.data_ptr() % 16 != 0
    assert all(torch.equal(a, b) for a, b in zip(gradients(q, k, v, odd, bits, None), want))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    radius_attention(*leaves, bits).sum().backward()
    ones = gradients(q, k, v, torch.ones_like(go), bits, None)
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, ones))


def test_gradient_against_differences(cuda):
    """Central differences of the float64 formula along random directions."""
    q, k, v, go, gen = operands(1, 2, 40, 32, torch.float16, 9, cuda)
    allowed = mask_of("random", 1, 40, gen)
    got = gradients(q, k, v, go, pack(allowed).to(cuda), None)
    _, _, _, bounds = reference(q, k, v, go, allowed, 32 ** -0.5)
    for i, name in enumerate(("q", "k", "v")):
        step = torch.randn(q.shape, generator=gen).to(cuda).double()
        ends = []
        for sign in (1e-4, -1e-4):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + sign * step
            ends.append(float((reference(*x, go, allowed, 32 ** -0.5)[0] * go.double()).sum()))
        slope = float((got[i].double() * step).sum())
        slack = float(((bounds[i] + got[i].double().abs() * 2.0 ** -11 + 2.0 ** -25) * step.abs()).sum())
        # the differences' own error: third derivatives times 1e-8, below 1e-6 of sums of order 10
        assert abs((ends[0] - ends[1]) / 2e-4 - slope) <= slack + 1e-5, name


def test_no_gradient_call_is_unchanged(cuda):
    q, k, v, _, gen = operands(1, 2, 90, 64, torch.bfloat16, 10, cuda)
    bits = pack(mask_of("random", 1, 90, gen)).to(cuda)
    plain = radius_attention(q, k, v, bits)
    tracked = radius_attention(q.detach().requires_grad_(True), k, v, bits)
    assert torch.equal(plain, tracked) and tracked.requires_grad and not plain.requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_stream_and_graph(cuda, dtype):
    q, k, v, go, gen = operands(2, 2, 130, 64, dtype, 11, cuda)
    bits = pack(mask_of("ragged", 2, 130, gen)).to(cuda)
    want = gradients(q, k, v, go, bits, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gradients(q, k, v, go, bits, None)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = gradients(q, k, v, go, bits, None)
    for turn in range(3):
        for t in (q, k, v, go):
            t.copy_(torch.randn(t.shape, generator=gen).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, gradients(q, k, v, go, bits, None))), turn


@pytest.mark.parametrize("N,block", [(1, False), (64, True), (100, False), (181, True), (300, True)])
def test_tables(cuda, N, block):
    gen = torch.Generator().manual_seed(N)
    allowed = mask_of("ragged" if N < 300 else "band", 2, N, gen)
    bm = blocks(allowed)
    if block and N > 64:  # a tile left out by the block mask is empty
        bm[1, 0, 1] = 0
        allowed[1, :64, 64:128] = False
    t = radius_tables(pack(allowed).to(cuda), bm.to(cuda) if block else None)
    NB = (N + 63) // 64
    full = torch.zeros(2, NB * 64, NB * 64, dtype=torch.bool)
    full[:, :N, :N] = allowed
    tiles = full.view(2, NB, 64, NB, 64)
    weight = torch.tensor([1 << i if i < 63 else -(1 << 63) for i in range(64)], dtype=torch.int64)
    assert torch.equal(t.bits_t.cpu(), pack(allowed.transpose(1, 2)))
    assert torch.equal(t.key_any.cpu(), (tiles.any(2) * weight).sum(-1))
    assert torch.equal(t.query_any.cpu(), (tiles.any(4).permute(0, 3, 1, 2) * weight).sum(-1))


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("scale", [0.2, -0.2])
@pytest.mark.parametrize("N", [100, 900])
def test_forward_with_tables(cuda, D, scale, N):
    """The tables change no finite result; with them atoms that are nobody's neighbour may hold NaN."""
    q, k, v, _, gen = operands(2, 2 if N < 900 else 80, N, D, torch.bfloat16, 12, cuda)
    allowed = mask_of("ragged", 2, N, gen)
    bits, bm = pack(allowed).to(cuda), blocks(allowed).to(cuda)
    tables = radius_tables(bits, bm)
    want = radius_attention(q, k, v, bits, bm, scale=scale, return_lse=True)
    got = radius_attention(q, k, v, bits, bm, scale=scale, return_lse=True, tables=tables)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    no_key, no_query = ~allowed.any(2).to(cuda), ~allowed.any(1).to(cuda)
    bad = [t.masked_fill(m[:, None, :, None], float("nan")) for t, m in zip((q, k, v), (no_key, no_query, no_query))]
    got = radius_attention(*bad, bits, bm, scale=scale, return_lse=True, tables=tables)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="radius_tables of this call"):
        radius_attention(q[:1], k[:1], v[:1], bits[:1], tables=tables)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [100, 300])
def test_large_finite_rows_without_a_partner_reach_nothing(cuda, dtype, N):
    """6e4 (near fp16's largest number) where nobody is paired: the scale of fp16's dS must not follow it."""
    q, k, v, go, gen = operands(2, 2, N, 64, dtype, 13, cuda)
    allowed = mask_of("ragged", 2, N, gen)
    bits = pack(allowed).to(cuda)
    no_key = ~allowed.any(2).to(cuda)[:, None, :]
    no_query = ~allowed.any(1).to(cuda)[:, None, :]
    assert no_key[1].any() and no_query[1].any()
    glse = torch.randn(2, 2, N, generator=gen).to(cuda)

    def grads(q, k, v, go, glse):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(radius_attention(*leaves, bits, return_lse=True), leaves, (go, glse))

    want = grads(q, k, v, go, glse)
    bad = [t.masked_fill(m[..., None], 6e4) for t, m in ((q, no_key), (k, no_query), (v, no_query), (go, no_key))]
    got = grads(*bad, glse.masked_fill(no_key, 1e30))
    for g, w, name in zip(got, want, ("dq", "dk", "dv")):
        assert torch.equal(g, w), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_keys_without_a_query_get_zeros_beside_a_row_that_is_not_finite(cuda, dtype):
    """Where a paired row's gradient is not finite, keys of its tile that nobody attends still get zeros."""
    q, k, v, go, gen = operands(1, 2, 60, 32, dtype, 14, cuda)
    allowed = mask_of("random", 1, 60, gen)
    allowed[:, :, [3, 40]] = False
    go[0, 1, 7, 5] = float("inf")
    dq, dk, dv = gradients(q, k, v, go, pack(allowed).to(cuda), None)
    for t in (dk, dv):
        assert torch.equal(t[:, :, [3, 40]], torch.zeros_like(t[:, :, [3, 40]]))


def test_value_gradients_of_keys_with_little_weight(cuda):
    """fp16: a key of weight 3e-9 in every row, gradients of 1e3: its dv of 1.2e-4 is within the type, though the weight
    by itself is below the type's smallest number.

    P is kept times 2^12, so what rounding it leaves is half a step: t relative, or 2^-25 2^-12 below the normal numbers;
    the logits here are sums of one exact product, so P's own error is the exponential's and lse's: 2^-20 + t + N u."""
    N, t = 40, 2.0 ** -11
    gen = torch.Generator().manual_seed(15)
    q = torch.zeros(1, 1, N, 32)
    k = torch.zeros(1, 1, N, 32)
    q[..., 0] = 4.0
    k[0, 0, 1, 0] = -4.0  # logit -16 against 0
    v = torch.randn(1, 1, N, 32, generator=gen)
    go = torch.randn(1, 1, N, 32, generator=gen).abs() * 1e3
    q, k, v, go = (x.to(torch.float16).to(cuda) for x in (q, k, v, go))
    allowed = torch.ones(1, N, N, dtype=torch.bool)
    got = gradients(q, k, v, go, pack(allowed).to(cuda), None, scale=1.0)[2]
    P = torch.softmax(q.double() @ k.double().mT, -1)
    want = P.mT @ go.double()
    slack = (P * (2 * t + 2 * N * U + 2.0 ** -20) + 2.0 ** -37).mT @ go.double().abs()
    assert float(want[0, 0, 1].min()) > 5e-5
    check(got, want, slack, "dv")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,D", [(70, 64), (30, 128), (129, 32), (128, 64)])
def test_tables_that_name_every_row(cuda, dtype, N, D):
    """Tables whose tiles are all marked, rows past the last atom too: the same gradients, none of those rows read."""
    from matterformer_amd.geometry_ops import RadiusTables

    q, k, v, go, gen = operands(2, 2, N, D, dtype, 16, cuda)
    allowed = mask_of("random", 2, N, gen)
    bits = pack(allowed).to(cuda)
    t = radius_tables(bits)
    every = RadiusTables(t.bits_t, torch.full_like(t.key_any, -1), torch.full_like(t.query_any, -1))
    want, got = gradients(q, k, v, go, bits, None, tables=t), gradients(q, k, v, go, bits, None, tables=every)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [65, 100, 192])
@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_head_dim_128_of_few_tiles_and_many_cells(cuda, dtype, N, scale):
    """Two and three tiles a cell, by the kernel of many workgroups and by that of few: each against float64, with and
    without tables, with NaN where nobody is paired, and the gradients of many.

    |out' - out| <= (2 es + 2 t + N u + 2^-20) sum P|v| + t |out| as above (P rounded, the sum, the last rounding)."""
    t = torch.finfo(dtype).eps / 2
    for B, H in ((40, 8), (3, 2)):
        q, k, v, go, gen = operands(B, H, N, 128, dtype, 17, cuda)
        allowed = mask_of("ragged", B, N, gen)
        bits = pack(allowed).to(cuda)
        tables = radius_tables(bits)
        out = radius_attention(q, k, v, bits, scale=scale)
        assert torch.equal(radius_attention(q, k, v, bits, scale=scale, tables=tables), out)
        want, _, grads, bounds = reference(q, k, v, go, allowed, scale)
        Q, K, V, A = q.double(), k.double(), v.double(), allowed.to(cuda)[:, None]
        s = (scale * (Q @ K.mT)).masked_fill(~A, -math.inf)
        P = torch.nan_to_num(torch.softmax(s, -1))
        es = 132 * U * abs(scale) * torch.where(A, Q.abs() @ K.abs().mT, 0.0).amax(-1, keepdim=True)
        check(out, want, (2 * es + 2 * t + N * U + 2.0 ** -20) * (P @ V.abs()), "out")
        no_key, no_query = ~allowed.any(2).to(cuda), ~allowed.any(1).to(cuda)
        bad = [x.masked_fill(m[:, None, :, None], float("nan")) for x, m in zip((q, k, v), (no_key, no_query, no_query))]
        assert torch.equal(radius_attention(*bad, bits, scale=scale, tables=tables), out)
        assert torch.equal(radius_attention(bad[0], k, v, bits, scale=scale), out)
        for g, w, b, name in zip(gradients(q, k, v, go, bits, None, scale=scale), grads, bounds, ("dq", "dk", "dv")):
            check(g, w, b, name)


@pytest.mark.parametrize("B,H,N", [(0, 2, 5), (2, 0, 5), (2, 2, 0)])
def test_empty(cuda, B, H, N):
    bits = torch.zeros(B, N, (N + 31) // 32, dtype=torch.int32, device=cuda)
    leaves = [torch.zeros(B, H, N, 32, dtype=torch.bfloat16, device=cuda, requires_grad=True) for _ in range(3)]
    with torch.no_grad():
        out, lse, out32 = radius_attention(*leaves, bits, return_lse=True, return_fp32=True)
    assert out.shape == (B, H, N, 32) and lse.shape == (B, H, N) and out32.dtype == torch.float32
    out = radius_attention(*leaves, bits)
    grads = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert all(g.shape == t.shape for g, t in zip(grads, leaves))
