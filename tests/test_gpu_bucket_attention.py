"""mf_bucket_attn and mf_bucket_attn_bwd against the formulas in 64 bits (tests/bucket_reference.py)."""

import math

import pytest
import torch

from matterformer_amd.bucket_attention import bucket_attention
from matterformer_amd.pair_buckets import MASKED, index_buckets, offset_buckets, offset_edges
from tests.bucket_reference import attention, check

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def gen_of(cuda, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def make(cuda, B, H, KV, Nq, Nk, D, dtype, *, K=17, mask="none", table=FP32, seed=0, batch=None):
    """q, k, v, table, index (uint8), go."""
    g = gen_of(cuda, seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda)
    q, k, v, go = (rnd(B, h, n, D).to(dtype) for h, n in ((H, Nq), (KV, Nk), (KV, Nk), (H, Nq)))
    batch = B if batch is None else batch
    index = torch.randint(0, K, (batch, Nq, Nk), generator=g, device=cuda, dtype=torch.int32)
    if mask == "holes":  # pairs left out at random, a query and a key without a pair
        index[torch.rand(index.shape, generator=g, device=cuda) < 0.5] = -1
        index[0, Nq // 2] = -1
        index[-1, :, Nk // 3] = -1
    elif mask == "padding":  # what padding holds reaches nothing
        for b in range(batch):
            cut_q, cut_k = max(1, Nq - 7 * b - 3), max(1, Nk - 13 * b - 5)
            index[b, cut_q:], index[b, :, cut_k:] = -1, -1
            q[b, :, cut_q:], go[b, :, cut_q:] = math.nan, math.inf
            k[b, :, cut_k:], v[b, :, cut_k:] = math.nan, -math.inf
    elif mask == "blocks":  # whole tiles without a pair
        i, j = (torch.arange(n, device=cuda) // 64 for n in (Nq, Nk))
        index[:, (i[:, None] + j[None]) % 3 != 0] = -1
    elif mask == "all":
        index.fill_(-1)
    return q, k, v, rnd(K, H).to(table), index, go


def run(q, k, v, table, index, go, *, glse=None, scale=None, K=None):
    buckets = index_buckets(index, table.shape[0])
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, table)]
    out, lse = bucket_attention(*leaves, buckets, scale=scale, return_lse=True)
    ups = (go,) if glse is None else (go, glse)
    grads = torch.autograd.grad((out,) if glse is None else (out, lse), leaves, ups)
    return dict(zip(("out", "lse", "dq", "dk", "dv", "dtable"), (out.detach(), lse.detach(), *grads)))


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 4, 4, 29, 29, 48), (2, 8, 2, 1, 300, 64), (1, 4, 1, 33, 65, 128), (2, 4, 4, 181, 181, 64),
          (1, 2, 2, 64, 128, 32), (1, 8, 8, 130, 257, 96), (3, 2, 1, 5, 1000, 40), (1, 12, 4, 100, 700, 128),
          (1, 2, 2, 257, 64, 24), (5, 3, 3, 19, 19, 64), (1, 1, 1, 500, 3, 16)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("mask", ["none", "holes", "padding", "blocks"])
@pytest.mark.parametrize("shape", SHAPES)
def test_output_and_gradients(cuda, shape, mask, dtype):
    B, H, KV, Nq, Nk, D = shape
    q, k, v, table, index, go = make(cuda, *shape, dtype, mask=mask, seed=sum(shape))
    r, bound = attention(q, k, v, table, index_buckets(index, table.shape[0]).index, D ** -0.5, go)
    check(run(q, k, v, table, index, go), r, bound)
    # without gradients: the same bits
    plain, lse = bucket_attention(q, k, v, table, index_buckets(index, table.shape[0], gradients=False), return_lse=True)
    check({"out": plain, "lse": lse}, r, bound)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 130, 64), (1, 6, 6, 29, 29, 32)])
def test_gradient_through_lse(cuda, shape, dtype):
    q, k, v, table, index, go = make(cuda, *shape, dtype, mask="holes")
    glse = torch.randn(shape[0], shape[1], shape[3], device=cuda) * 3.0
    buckets = index_buckets(index, table.shape[0])
    r, bound = attention(q, k, v, table, buckets.index, shape[-1] ** -0.5, go, glse)
    check(run(q, k, v, table, index, go, glse=glse), r, bound)
    # lse alone
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, table)]
    _, lse = bucket_attention(*leaves, buckets, return_lse=True)
    grads = torch.autograd.grad(lse, leaves, glse)
    r, bound = attention(q, k, v, table, buckets.index, shape[-1] ** -0.5, torch.zeros_like(go), glse)
    check(dict(zip(("dq", "dk", "dv", "dtable"), grads)), r, bound)
    assert not grads[2].any()


@pytest.mark.parametrize("table_dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("K", [1, 2, 32, 63, 64])
def test_tables(cuda, K, table_dtype):
    q, k, v, table, index, go = make(cuda, 2, 4, 2, 100, 70, 64, BF16, K=K, table=table_dtype)
    r, bound = attention(q, k, v, table, index_buckets(index, K).index, 0.125, go)
    check(run(q, k, v, table, index, go), r, bound)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-30])
def test_scales(cuda, scale):
    q, k, v, table, index, go = make(cuda, 1, 2, 2, 70, 90, 32, BF16)
    r, bound = attention(q, k, v, table, index_buckets(index, table.shape[0]).index, scale, go)
    check(run(q, k, v, table, index, go, scale=scale), r, bound)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Nq", [1, 40, 200])
def test_entries_of_minus_infinity(cuda, dtype, Nq):
    """A bucket whose bias is -inf leaves its pairs out; a row that has no other gives 0, and takes no gradient."""
    q, k, v, table, index, go = make(cuda, 2, 4, 2, Nq, 150, 64, dtype, K=5)
    table[2] = -math.inf
    table[3, 1] = -math.inf
    index[0, Nq // 2] = 2
    index[1, 0] = 3
    buckets = index_buckets(index, 5)
    r, bound = attention(q, k, v, table, buckets.index, 0.125, go)
    got = run(q, k, v, table, index, go)
    check(got, r, bound)
    assert not got["out"][0, :, Nq // 2].any() and not got["lse"][0, :, Nq // 2].any() and not got["dq"][0, :, Nq // 2].any()
    assert not got["dtable"][2].any() and got["dtable"][3, 1] == 0


@pytest.mark.parametrize("low", [-1e4, -65504.0, -1e9, torch.finfo(BF16).min, torch.finfo(FP32).min])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_finite_mask_values(cuda, low, dtype):
    """A huge negative bias masks beside others; a row that has nothing else is an average of what its rounding leaves, as a
    softmax over it alone is: of all keys alike once the value swallows the products."""
    q, k, v, table, index, go = make(cuda, 1, 2, 2, 40, 100, 64, dtype, K=4)
    table[1] = low
    index[0, 5] = 1
    index[0, 6] = 1
    index[0, 6, 70:] = -1
    buckets = index_buckets(index, 4)
    got = run(q, k, v, table, index, go)
    assert all(torch.isfinite(t).all() for t in got.values())
    q2, go2, index2 = q.clone(), go.clone(), index.clone()
    rest = [i for i in range(40) if i not in (5, 6)]
    r, bound = attention(q2[:, :, rest].contiguous(), k, v, table.clamp_min(-3e38), index_buckets(index2[:, rest], 4).index, 0.125,
                         go2[:, :, rest].contiguous())
    check({n: got[n][:, :, rest] for n in ("out", "dq")}, r, bound)
    if low < -1e8:
        # x - m is 0 for every pair of the row but where a step of x is small beside the products: below -2^27 none is
        for i, keys in ((5, 100), (6, 70)):
            mean = v[0, :, :keys].double().mean(1)
            off = (got["out"][0, :, i].double() - mean).abs()
            assert (off <= (2 * 2.0 ** -9 if dtype == BF16 else 2 * 2.0 ** -12) * v[0].double().abs().amax(1) + 2.0 ** -8 * mean.abs()).all()


def test_head_layouts_and_strides(cuda):
    """Views of projected rows, sliced, transposed, misaligned and broadcast operands give what contiguous ones give, and
    gradients in the operands' layout."""
    B, N, H, KV, D = 2, 90, 4, 2, 48
    g = gen_of(cuda, 4)
    rows = torch.randn(B, N, (H + 2 * KV) * D, generator=g, device=cuda).to(BF16)
    table = torch.randn(9, H, generator=g, device=cuda)
    index = torch.randint(0, 9, (B, N, N), generator=g, device=cuda)
    buckets = index_buckets(index, 9)
    go = torch.randn(B, N, H, D, generator=g, device=cuda).to(BF16).transpose(1, 2)

    def heads(r):
        q, k, v = r.split((H * D, KV * D, KV * D), dim=-1)
        return [t.view(B, N, -1, D).transpose(1, 2) for t in (q, k, v)]

    leaf = rows.clone().requires_grad_(True)
    out = bucket_attention(*heads(leaf), table, buckets)
    (grad,) = torch.autograd.grad(out, leaf, go)
    assert out.transpose(1, 2).is_contiguous()  # merged without a copy
    plain = [t.contiguous().requires_grad_(True) for t in heads(rows)]
    want = bucket_attention(*plain, table, buckets)
    dq, dk, dv = torch.autograd.grad(want, plain, go.contiguous())
    assert torch.equal(out, want)
    assert torch.equal(grad, torch.cat([t.transpose(1, 2).flatten(2) for t in (dq, dk, dv)], dim=-1))

    q, k, v = (t.contiguous() for t in heads(rows))
    for change in (lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),  # entries apart
                   lambda t: torch.cat([t, t], dim=2)[:, :, :N],              # a slice
                   lambda t: torch.cat([t, t], dim=3)[..., 8:8 + D].contiguous().flatten().clone().view_as(t),
                   lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view_as(t).copy_(t)):  # misaligned
        args = [change(t) for t in (q, k, v)]
        fixed = [t.contiguous() for t in args]
        assert torch.equal(bucket_attention(*args, table, buckets), bucket_attention(*fixed, table, buckets))
    one = q[:1, :1].requires_grad_(True)
    wide = bucket_attention(one.expand(B, H, N, D), k, v, table, buckets)
    (summed,) = torch.autograd.grad(wide, one, go)
    full = one.detach().expand(B, H, N, D).contiguous().requires_grad_(True)
    (each,) = torch.autograd.grad(bucket_attention(full, k, v, table, buckets), full, go)
    assert torch.equal(summed, each.sum((0, 1), keepdim=True))
    # a gradient that is a broadcast view
    (ones,) = torch.autograd.grad(bucket_attention(full, k, v, table, buckets).sum(), full)
    (same,) = torch.autograd.grad(bucket_attention(full, k, v, table, buckets), full, torch.ones_like(full))
    assert torch.equal(ones, same)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_buckets_of_one_entry_serve_a_batch(cuda, dtype):
    q, k, v, table, index, go = make(cuda, 3, 4, 4, 100, 100, 32, dtype, mask="holes", batch=1)
    r, bound = attention(q, k, v, table, index_buckets(index, table.shape[0]).index, 32 ** -0.5, go)
    check(run(q, k, v, table, index, go), r, bound)


@pytest.mark.parametrize("B,H,KV,Nq,Nk,D", [(1, 8, 8, 1, 5000, 64), (2, 12, 3, 1, 3001, 128), (1, 32, 1, 1, 700, 64),
                                            (1, 32, 1, 4, 900, 32), (4, 4, 4, 3, 20000, 32), (1, 2, 1, 64, 4100, 128)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_few_queries_over_long_caches(cuda, B, H, KV, Nq, Nk, D, dtype):
    """New tokens: positions at the end of caches of different lengths, what lies behind them is anything."""
    g = gen_of(cuda, Nk)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    q, k, v = rnd(B, H, Nq, D), rnd(B, KV, Nk, D), rnd(B, KV, Nk, D)
    length = torch.randint(Nq, Nk + 1, (B, 1), generator=g, device=cuda)
    length[0] = Nk
    pad = torch.arange(Nk, device=cuda)[None] >= length
    k.masked_fill_(pad[:, None, :, None], math.nan)
    v.masked_fill_(pad[:, None, :, None], math.inf)
    places = length - Nq + torch.arange(Nq, device=cuda)[None]
    buckets = offset_buckets(places, torch.arange(Nk, device=cuda), offset_edges(32, 512, causal=True), pad_mask=pad,
                             causal=True, gradients=False)
    table = torch.randn(32, H, generator=g, device=cuda)
    out, lse = bucket_attention(q, k, v, table, buckets, return_lse=True)
    r, bound = attention(q, k, v, table, buckets.index, D ** -0.5)
    check({"out": out, "lse": lse}, r, bound)
    assert torch.equal(out, bucket_attention(q, k, v, table, buckets))


def test_small_weights_beside_a_large_one(cuda):
    """fp16: 131072 keys of weight 2^-25 beside one of weight 1 are 0.4 % of the row, not nothing."""
    Nk = 131073
    q = torch.ones(1, 1, 1, 8, device=cuda, dtype=FP16)
    k, v = torch.zeros(1, 1, Nk, 8, device=cuda, dtype=FP16), torch.ones(1, 1, Nk, 8, device=cuda, dtype=FP16)
    v[:, :, 0] = 0
    index = torch.ones(1, 1, Nk, dtype=torch.int32, device=cuda)
    index[..., 0] = 0
    table = torch.tensor([[25.0 * math.log(2.0)], [0.0]], device=cuda)
    out = bucket_attention(q, k, v, table, index_buckets(index, 2, gradients=False))
    want = 131072 * 2.0 ** -25 / (1 + 131072 * 2.0 ** -25)
    assert (out.double() - want).abs().max() <= want * (2.0 ** -11 * 2 + 2.0 ** -15)


def test_caches_past_2_31_elements(cuda):
    """k and v of 2.2e9 elements each, the last request's rows past 2^31."""
    B, KV, Nk, D = 17, 8, 131072, 128
    k = torch.empty(B, KV, Nk, D, device=cuda, dtype=BF16)
    v = torch.empty_like(k)
    g = gen_of(cuda, 9)
    for b in (0, B - 1):
        k[b] = torch.randn(KV, Nk, D, generator=g, device=cuda).to(BF16)
        v[b] = torch.randn(KV, Nk, D, generator=g, device=cuda).to(BF16)
    k[1:-1], v[1:-1] = 0, 0
    q = torch.randn(B, KV, 1, D, generator=g, device=cuda).to(BF16)
    places = torch.arange(Nk, device=cuda)
    buckets = offset_buckets(places[-1:], places, offset_edges(16, 1000, causal=True), causal=True, gradients=False)
    table = torch.randn(16, KV, generator=g, device=cuda)
    out = bucket_attention(q, k, v, table, buckets)
    assert k.numel() > 2 ** 31
    for b in (0, B - 1):
        r, bound = attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], table, buckets.index, D ** -0.5)
        check({"out": out[b:b + 1]}, r, bound)


def test_two_calls_give_identical_bits(cuda):
    q, k, v, table, index, go = make(cuda, 3, 8, 2, 200, 333, 64, FP16, mask="holes")
    a, b = run(q, k, v, table, index, go), run(q, k, v, table, index, go)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_empty_calls(cuda):
    for B, H, Nq, Nk in ((0, 2, 5, 5), (2, 0, 5, 5), (2, 2, 0, 5), (2, 2, 5, 0)):
        q = torch.randn(B, H, Nq, 32, device=cuda, dtype=BF16, requires_grad=True)
        k, v = (torch.randn(B, H, Nk, 32, device=cuda, dtype=BF16, requires_grad=True) for _ in range(2))
        table = torch.randn(4, H, device=cuda, requires_grad=True)
        out, lse = bucket_attention(q, k, v, table, index_buckets(torch.zeros(B, Nq, Nk, dtype=torch.int32, device=cuda), 4),
                                    return_lse=True)
        assert out.shape == q.shape and not out.any() and lse.shape == q.shape[:3] and not lse.any()
        grads = torch.autograd.grad(out, (q, k, v, table), torch.ones_like(out))
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v, table)))


def test_nobody_pairs(cuda):
    q, k, v, table, index, go = make(cuda, 2, 4, 2, 70, 90, 64, BF16, mask="all")
    q[:], k[:], v[:], go[:] = math.nan, math.inf, math.nan, math.nan
    assert all(not t.any() for t in run(q, k, v, table, index, go).values())


def test_differences(cuda):
    """The gradients against differences of the kernel's own output: the loss is summed in 64 bits, and steps in which the
    output's rounding is small are taken along the gradient."""
    q, k, v, table, index, go = make(cuda, 1, 2, 1, 64, 64, 32, FP16, K=8)
    got = run(q, k, v, table, index, go)
    buckets = index_buckets(index, 8)
    loss = lambda *a: (bucket_attention(*a, buckets).double() * go.double()).sum().item()
    for n, name in ((3, "dtable"),):
        args = [q, k, v, table]
        direction = got[name].double()
        h = 0.05 / direction.abs().max().item()
        up, down = ((table.double() + s * h * direction).float() for s in (1, -1))
        slope = (loss(q, k, v, up) - loss(q, k, v, down)) / (2 * h)
        want = direction.square().sum().item()
        # a rounding of every output entry, random in sign: 2^-12 of |out| <= 4 by |go| <= 4 over sqrt(entries), by 2 h
        noise = 2.0 ** -12 * (go.double().square().sum().sqrt().item()) * 4 / h
        assert abs(slope - want) <= 0.02 * want + noise


def test_refused_calls(cuda):
    b = index_buckets(torch.zeros(2, 3, 5, dtype=torch.int32, device=cuda), 4)
    q, k, table = (torch.zeros(*s, device=cuda) for s in ((2, 4, 3, 8), (2, 2, 5, 8), (4, 4)))
    h = lambda t: t.to(BF16)
    for args, match in (((q, k, k, table, b), "float16/bfloat16"), ((h(q), h(k), h(k).half(), table, b), "one dtype"),
                        ((h(q), h(k), h(k), table.double(), b), "table"), ((h(q).cpu(), h(k), h(k), table, b), "same device"),
                        ((h(q)[..., :4], h(k)[..., :4], h(k)[..., :4], table, b), "multiples of 8"),
                        ((h(q).repeat(1, 17, 1, 1), h(k), h(k), table.repeat(1, 17), b), "up to 32 heads")):
        with pytest.raises(RuntimeError, match=match):
            bucket_attention(*args)
    wide = torch.zeros(2, 4, 3, 136, device=cuda, dtype=BF16)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        bucket_attention(wide, wide[:, :2, :1].expand(2, 2, 5, 136), wide[:, :2, :1].expand(2, 2, 5, 136), table, b)
    once = index_buckets(torch.zeros(2, 3, 5, dtype=torch.int32, device=cuda), 4, gradients=False)
    with pytest.raises(ValueError, match="gradients=True"):
        bucket_attention(h(q).requires_grad_(True), h(k), h(k), table, once)


def test_another_stream(cuda):
    q, k, v, table, index, go = make(cuda, 2, 8, 8, 300, 300, 64, BF16, mask="holes")
    want = run(q, k, v, table, index, go)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run(q, k, v, table, index, go))
    torch.cuda.synchronize()
    assert all(torch.equal(want[n], g[n]) for g in got for n in want)


@pytest.mark.parametrize("shape", [(2, 4, 2, 100, 130, 64), (1, 8, 2, 1, 3000, 64)])
def test_replayed_graph(cuda, shape):
    q, k, v, table, index, go = make(cuda, *shape, BF16)
    buckets = index_buckets(index, table.shape[0])
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, table)]

    def step():
        out = bucket_attention(*leaves, buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(step())
    for n in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn_like(t))
        want = step()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for mine in held:
            assert all(torch.equal(a, b) for a, b in zip(mine, want))


def test_saved_tensors_moved_meanwhile(cuda):
    """Saved tensor hooks hand the backward pass other tensors than the forward saw."""
    B, N, H, D = 2, 80, 4, 64
    rows = torch.randn(B, N, 3 * H * D, device=cuda).to(BF16).requires_grad_(True)
    q, k, v = (t.view(B, N, H, D).transpose(1, 2) for t in rows.chunk(3, dim=-1))
    table = torch.randn(8, H, device=cuda, requires_grad=True)
    buckets = index_buckets(torch.randint(0, 8, (B, N, N), device=cuda), 8)
    go = torch.randn(B, H, N, D, device=cuda).to(BF16)
    want = torch.autograd.grad(bucket_attention(q, k, v, table, buckets), (rows, table), go)
    with torch.autograd.graph.save_on_cpu():
        out = bucket_attention(*(t.view(B, N, H, D).transpose(1, 2) for t in rows.chunk(3, dim=-1)), table, buckets)
    got = torch.autograd.grad(out, (rows, table), go)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_buckets_made_in_inference_mode(cuda):
    q, k, v, table, index, go = make(cuda, 1, 2, 2, 40, 40, 32, BF16)
    with torch.inference_mode():
        buckets = index_buckets(index, table.shape[0])
        plain = bucket_attention(q, k, v, table, buckets)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, table)]
    out = bucket_attention(*leaves, buckets)
    assert torch.equal(out, plain)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(out, leaves, go))


def test_two_layers_share_buckets_and_a_table(cuda):
    """One table through two layers: its gradient is the sum of both."""
    q, k, v, table, index, go = make(cuda, 2, 4, 4, 70, 70, 32, BF16)
    buckets = index_buckets(index, table.shape[0])
    t = table.clone().requires_grad_(True)
    first = bucket_attention(q, k, v, t, buckets)
    both = first + bucket_attention(v, k, q, t, buckets)
    (together,) = torch.autograd.grad(both, t, go)
    each = [torch.autograd.grad(bucket_attention(a, k, c, t, buckets), t, go)[0] for a, c in ((q, v), (v, q))]
    assert torch.allclose(together, each[0] + each[1], rtol=1e-6, atol=1e-6)


def test_forward_mode_is_refused(cuda):
    from torch.autograd import forward_ad

    q, k, v, table, index, _ = make(cuda, 1, 2, 2, 20, 20, 32, BF16)
    buckets = index_buckets(index, table.shape[0])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            bucket_attention(dual, k, v, table, buckets)


def backward_plan(B, H, KV, Nq, Nk, D, dtype, K):
    """(pieces, row tiles a piece) of the queries' and of the keys' kernel, as csrc/bucket_attn_bwd.hip takes them; held
    against the workspace that the library asks for."""
    from matterformer_amd import _native

    DP = 32 if D <= 32 else 64 if D <= 64 else 128
    TQ, TK = (-(-n // 64) for n in (Nq, Nk))

    def side(batch_heads, columns, tiles, keys):
        W = 1 if columns <= 32 else 2 if columns <= 64 else 4
        CT = -(-columns // (32 * W))
        units, room = batch_heads * CT, 1024 * (1 if keys and DP == 128 else 2)
        pieces = max(1, min(tiles, room // max(1, units * W)))
        per_piece = -(-tiles // pieces)
        pieces = -(-tiles // per_piece)
        split = units * pieces * 32 * W * (2 * DP if keys else DP + 1) * 4 if pieces > 1 else 0
        return CT, pieces, per_piece, split

    queries, keys = side(B * H, Nq, TK, False), side(B * KV, Nk, H // KV * TQ, True)
    up = lambda n: -(-n // 256) * 256
    nbytes = up(B * H * TQ * 3 * 64 * 4) + up(H * K * B * keys[0] * keys[1] * 4) + up(max(queries[3], keys[3]))
    if dtype == FP16:
        nbytes += up((B * H * TQ + B * KV * TK) * 16)
    args = _native.MfBucketAttnBwdArgs(dtable=16, fwd=_native.MfBucketAttnArgs(
        batch=B, heads=H, kv_heads=KV, queries=Nq, keys=Nk, head_dim=D, buckets=K, dtype=_native.dtype_code(dtype)))
    assert _native.lib().mf_bucket_attn_bwd_workspace_size(args) == nbytes
    return queries[1:3], keys[1:3]


# (shape, type, mask, pieces and row tiles a piece of the queries' and the keys' kernel): workgroups that stream many tiles,
# through several heads, in one piece and in pieces that begin within a head
STREAMED = [((32, 8, 8, 512, 512, 64), BF16, "none", (1, 8), (1, 8)), ((32, 8, 8, 512, 512, 64), FP16, "holes", (1, 8), (1, 8)),
            ((64, 8, 8, 181, 181, 64), BF16, "padding", (1, 3), (1, 3)), ((64, 8, 2, 300, 181, 128), FP16, "padding", (1, 3), (1, 20)),
            ((4, 8, 2, 1300, 1300, 64), BF16, "holes", (1, 21), (5, 17)), ((4, 8, 2, 1997, 1997, 128), FP16, "none", (1, 32), (2, 64)),
            ((4, 8, 2, 1997, 1997, 128), BF16, "blocks", (1, 32), (2, 64)), ((40, 16, 4, 700, 60, 32), BF16, "holes", (1, 1), (6, 8)),
            ((4, 4, 1, 500, 3000, 64), FP16, "holes", (8, 6), (5, 7)),
            ((40, 32, 8, 20, 700, 32), FP16, "holes", (1, 11), (1, 4)), ((16, 32, 32, 130, 400, 24), BF16, "blocks", (1, 7), (1, 3))]


@pytest.mark.parametrize("shape,dtype,mask,queries,keys", STREAMED, ids=lambda x: str(x).replace(" ", "") if isinstance(x, tuple) else None)
def test_workgroups_that_stream_many_tiles(cuda, shape, dtype, mask, queries, keys):
    q, k, v, table, index, go = make(cuda, *shape, dtype, K=32, mask=mask, seed=sum(shape))
    assert backward_plan(*shape, dtype, 32) == (queries, keys)
    got = run(q, k, v, table, index, go)
    # batch entries have rows of their own; only the table's gradient joins them
    total, most = 0.0, 0.0
    per = max(1, 2 ** 27 // (shape[1] * shape[3] * shape[4]))
    for b in range(0, shape[0], per):
        at = slice(b, b + per)
        r, bound = attention(q[at], k[at], v[at], table, index_buckets(index[at], 32).index, shape[5] ** -0.5, go[at])
        check({n: got[n][at] for n in ("out", "lse", "dq", "dk", "dv")}, r, bound)
        total, most = total + r["dtable"], most + bound["dtable"]
    check({"dtable": got["dtable"]}, {"dtable": total}, {"dtable": most})


@pytest.mark.parametrize("shape,dtype", [((2, 6, 3, 1500, 1500, 64), FP16), ((1, 4, 4, 2100, 2100, 128), BF16),
                                         ((1, 12, 6, 1100, 1600, 32), BF16), ((3, 4, 2, 1700, 1200, 96), FP16)])
def test_earlier_keys_of_few_heads(cuda, shape, dtype):
    """Fewer than eight key heads in all and more than eight tiles: the tiles are dealt in eight sequences."""
    B, H, KV, Nq, Nk, D = shape
    assert B * KV < 8 and min(Nq, Nk) > 8 * 128
    q, k, v, table, _, go = make(cuda, *shape, dtype, K=32, seed=sum(shape))
    places = [torch.arange(n, device=cuda) for n in (Nq, Nk)]
    buckets = offset_buckets(*places, offset_edges(32, 900, causal=True), causal=True)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, table)]
    out, lse = bucket_attention(*leaves, buckets, return_lse=True)
    grads = torch.autograd.grad(out, leaves, go)
    got = dict(zip(("out", "lse", "dq", "dk", "dv", "dtable"), (out.detach(), lse.detach(), *grads)))
    r, bound = attention(q, k, v, table, buckets.index, D ** -0.5, go)
    check(got, r, bound)


@pytest.mark.parametrize("low", [-1e9, torch.finfo(BF16).min, torch.finfo(FP32).min])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Nq", [40, 200])
def test_gradients_of_rows_at_finite_mask_values(cuda, low, dtype, Nq):
    """Rows all of whose biases are huge and negative: x is the bias alone (its fp32 step, 128 in log2 units at least, swallows
    the products), so that P is 1 over the number of pairs, exactly alike."""
    B, H, Nk, D, scale = 2, 2, 100, 64, 0.125
    q, k, v, table, index, go = make(cuda, B, H, H, Nq, Nk, D, dtype, K=4)
    table[1] = low
    rows = {5: Nk, 6: 70, Nq - 1: Nk}
    for i in rows:
        index[0, i] = 1
    index[0, 6, 70:] = -1
    got = run(q, k, v, table, index, go)
    # in 64 bits their products would count: with queries of zeros there they do not, and dk's part of them is added
    flat = q.clone()
    flat[0, :, list(rows)] = 0
    codes = index_buckets(index, 4).index
    r, bound = attention(flat, k, v, table.clamp_min(-1e9), codes, scale, go)
    u, f = torch.finfo(dtype).eps / 2, 2.0 ** -15
    grain = 2.0 ** -25 if dtype == FP16 else 0.0
    g64, q64, v64 = go.double(), q.double(), v.double()
    peak = 2.0 * g64.norm(dim=-1).max() * v64.norm(dim=-1).max()
    for i, n in rows.items():
        vi, g = v64[0, :, :n], g64[0, :, i]  # (H, n, D), (H, D)
        dP = (vi @ g[..., None])[..., 0]
        out = vi.mean(1)
        dS = (dP - (out * g).sum(-1, keepdim=True)) / n
        spread = vi.abs().mean(1)
        wide = (g.abs() * (out.abs() + spread * (u + f))).sum(-1, keepdim=True)
        off = ((vi.abs() @ g.abs()[..., None])[..., 0] + wide) * f / n
        dS_off = dS.abs() * u + off + grain * peak * 2.0 ** -12
        r["dk"][0, :, :n] += scale * dS[..., None] * q64[0, :, i, None]
        bound["dk"][0, :, :n] += scale * dS_off[..., None] * q64[0, :, i, None].abs() + u * scale * (dS[..., None] * q64[0, :, i, None]).abs()
    r.pop("lse")  # (beside the bias its 64-bit value has more bits than fp32)
    check({n: got[n] for n in r}, r, bound)
    # and their outputs are the plain means
    for i, n in rows.items():
        mean = v64[0, :, :n].mean(1)
        assert ((got["out"][0, :, i].double() - mean).abs() <= bound["out"][0, :, i]).all()


@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 700, 64), (1, 8, 2, 1, 3000, 64), (16, 8, 8, 300, 300, 32)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_statistics_for_the_gradients(cuda, dtype, shape):
    """The pairs (a, c) that the forward leaves, also where a row's maximum rises slowly from tile to tile or is huge:
    P = 2^(log2(e) S - a) c and log2(e) S - a < 1, zeros for a row without a pair."""
    from matterformer_amd.bucket_attention import _forward

    B, H, KV, Nq, Nk, D = shape
    q, k, v, table, index, _ = make(cuda, *shape, dtype, K=17, mask="holes")
    index[-1, 0] = 16
    table[16] = -1e9
    k *= torch.linspace(0.1, 3.0, Nk, device=cuda).to(dtype)[:, None]
    buckets = index_buckets(index, 17)
    stats = _forward(q, k, v, table, buckets, D ** -0.5, lse=True, training=True)[3]
    a, c = stats.double()[..., None].unbind(0)
    allowed = (buckets.index != MASKED)[:, None]
    wide = torch.cat([table.double(), table.new_zeros(1, H).double()])[torch.where(buckets.index == MASKED, 17, buckets.index).long()]
    s = q.double() @ k.double().repeat_interleave(H // KV, 1).transpose(-1, -2).contiguous() * D ** -0.5 + wide.permute(0, 3, 1, 2)
    x = torch.where(allowed, s * math.log2(math.e), -math.inf)
    # fp32 roundings of x: of a few hundred at most by 2^-24 a term; of the huge row all of the products
    slack = torch.where(x.amax(-1, keepdim=True) < -1e6, 300.0, 2.0 ** -12)
    assert ((x - a < 1.0 + slack) | ~allowed).all()
    P = torch.softmax(torch.where(allowed, s, -math.inf), -1)
    some = allowed.any(-1, keepdim=True) & (x.amax(-1, keepdim=True) > -1e6)
    off = (torch.exp2(x - a) * c - P).abs()
    assert ((off <= 2.0 ** -12 * P) | ~(allowed & some)).all()
    none = ~allowed.any(-1, keepdim=True).expand_as(a)
    assert not a[none].any() and not c[none].any()
    huge = (a < -1e6)
    assert huge.any() and (c[huge] - 1.0 / allowed.expand(B, H, Nq, Nk).sum(-1, keepdim=True)[huge]).abs().max() <= 2.0 ** -20
