"""mf_pair_buckets, mf_bucket_bias and mf_bucket_bias_bwd on the GPU against the torch formulations on the CPU and 64-bit
sums."""

import math

import pytest
import torch

from matterformer_amd.pair_buckets import (MASKED, bucket_bias, distance_buckets, index_buckets, offset_buckets, offset_edges,
                                           value_buckets)
from tests.bucket_reference import dense, step

pytestmark = pytest.mark.gpu


def same(got, want):
    """The buckets of a GPU call and of the same call on the CPU, and what its tiles say of them."""
    torch.cuda.synchronize()
    B, Nq, Nk = want.index.shape
    assert got.num_buckets == want.num_buckets
    assert torch.equal(got.index.cpu(), want.index)
    if want.index_t is not None:
        assert torch.equal(got.index_t.cpu(), want.index_t)
    pad_q, pad_k = -Nq % 64, -Nk % 64
    on = torch.nn.functional.pad(want.index != MASKED, (0, pad_k, 0, pad_q))
    tiles = on.view(B, (Nq + pad_q) // 64, 64, (Nk + pad_k) // 64, 64)
    weights = torch.tensor([1 << t if t < 63 else -(1 << 63) for t in range(64)])
    assert torch.equal(got.key_any.cpu(), (tiles.any(2).long() * weights).sum(-1))
    assert torch.equal(got.query_any.cpu().transpose(1, 2), (tiles.any(4).long() * weights[:, None]).sum(2))
    # the bytes behind the last key are masked: a row is read whole
    for t, n in ((got.index, Nk), (got.index_t, Nq)):
        if t is not None and t.numel():
            whole = t.as_strided((*t.shape[:2], t.stride(1)), t.stride())
            assert whole[:, :, n:].eq(MASKED).all()


@pytest.mark.parametrize("B,N", [(1, 1), (3, 19), (2, 64), (2, 65), (5, 181), (1, 700)])
@pytest.mark.parametrize("edges,cutoff", [([], None), ([0.0, 1.0], None), ([0.3 * i for i in range(1, 64)], 9.0)])
def test_distance_buckets(cuda, B, N, edges, cutoff):
    g = torch.Generator().manual_seed(N)
    coords = torch.randn(B, N, 3, generator=g) * 4.0
    pad = torch.arange(N)[None] >= torch.randint(1, N + 1, (B, 1), generator=g)
    for mask in (None, pad):
        same(distance_buckets(coords.to(cuda), edges, pad_mask=None if mask is None else mask.to(cuda), cutoff=cutoff),
             distance_buckets(coords, edges, pad_mask=mask, cutoff=cutoff))


def test_distances_at_and_beside_edges(cuda):
    """Points on a lattice of eighths and a step of fp32 beside it: many distances equal an edge or miss it by a step."""
    g = torch.Generator().manual_seed(1)
    coords = torch.randint(-16, 17, (2, 150, 3), generator=g) / 8.0
    up = torch.nextafter(coords, torch.full_like(coords, math.inf))
    coords = torch.where(torch.rand(coords.shape, generator=g) < 0.2, up, coords)
    edges = [i / 8.0 for i in range(1, 40)]
    same(distance_buckets(coords.to(cuda), edges, cutoff=4.5), distance_buckets(coords, edges, cutoff=4.5))
    # exact: the squares' sums in whole numbers of 2^-46
    d = (coords[0, :, None].double() - coords[0, None].double()) * 2.0 ** 25
    ok = 0
    got = distance_buckets(coords.to(cuda), edges).index[0].cpu()
    for i in range(0, 150, 13):
        for j in range(0, 150, 7):
            square = sum(int(x) ** 2 for x in d[i, j].tolist())
            ok += int(got[i, j]) == sum(square >= (e * 2 ** 22) ** 2 for e in range(1, 40))
    assert ok == len(range(0, 150, 13)) * len(range(0, 150, 7))


def test_coordinates_that_are_not_finite_or_large(cuda):
    coords = torch.tensor([[[0.0, 0, 0], [math.nan, 0, 0], [math.inf, 0, 0], [-math.inf, 0, 0], [3e38, 3e38, 0], [-3e38, 0, 0]]])
    edges = [1.0, 1e30, 3e38]
    same(distance_buckets(coords.to(cuda), edges), distance_buckets(coords, edges))


@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 500), (70, 3), (130, 257), (64, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_offset_buckets(cuda, Nq, Nk, causal):
    g = torch.Generator().manual_seed(Nq + Nk)
    qp, kp = (torch.randint(-50, 2000, (3, n), generator=g) for n in (Nq, Nk))
    qpad, kpad = (torch.rand(3, n, generator=g) < 0.2 for n in (Nq, Nk))
    edges = offset_edges(33, 700)
    for q, k, gradients in ((qp, kp, True), (qp[0], kp, False), (qp.int(), kp[:1], True), (qp[0], kp[0], True)):
        masks = dict(pad_mask=kpad, query_pad_mask=qpad) if max(q.ndim, k.ndim) > 1 and k.shape[0] != 1 or q.ndim > 1 else {}
        on = {n: m.to(cuda) for n, m in masks.items()}
        same(offset_buckets(q.to(cuda), k.to(cuda), edges, causal=causal, gradients=gradients, **on),
             offset_buckets(q, k, edges, causal=causal, gradients=gradients, **masks))
    # a strided row of positions
    same(offset_buckets(qp.to(cuda).t().contiguous().t(), kp.to(cuda), edges, causal=causal),
         offset_buckets(qp, kp, edges, causal=causal))


def test_far_positions(cuda):
    p = torch.tensor([0, 1, 2 ** 31, 2 ** 31 + 1, 2 ** 53, 2 ** 53 + 1, 2 ** 61])
    edges = [-(2 ** 53), -1, 0, 1, 2, 2 ** 31, 2 ** 53]
    same(offset_buckets(p.to(cuda), p.to(cuda), edges), offset_buckets(p, p, edges))


@pytest.mark.parametrize("causal", [False, True])
def test_near_and_far_positions_in_one_tile(cuda, causal):
    """Rows whose queries are far from the tile's keys beside rows whose queries are near, padded ones among them."""
    g = torch.Generator().manual_seed(8)
    edges = offset_edges(24, 300)
    for first, last, shift in ((0, 16, 2 ** 40), (0, 16, -(2 ** 29)), (40, 60, 2 ** 29 - 3), (5, 6, -(2 ** 35))):
        qp, kp = torch.randint(0, 700, (2, 130), generator=g), torch.randint(0, 700, (2, 200), generator=g)
        qp[:, first:last] += shift
        kp[1, 70:90] += shift // 2
        pad, qpad = (torch.rand(2, n, generator=g) < 0.3 for n in (200, 130))
        masks = dict(pad_mask=pad, query_pad_mask=qpad)
        same(offset_buckets(qp.to(cuda), kp.to(cuda), edges, causal=causal, **{n: m.to(cuda) for n, m in masks.items()}),
             offset_buckets(qp, kp, edges, causal=causal, **masks))


@pytest.mark.parametrize("B,N", [(1, 300), (2, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_places_in_order(cuda, B, N, causal):
    """Tiles far from the diagonal, which have one bucket."""
    places = torch.arange(N)[None].expand(B, N) * 3
    pad = torch.arange(N)[None] >= torch.tensor([[N - 37 * b] for b in range(B)])
    for edges in ([], [0], offset_edges(9, 40), [-10 ** 6, -400, 5, 399, 10 ** 6]):
        same(offset_buckets(places.to(cuda), places.to(cuda), edges, pad_mask=pad.to(cuda), query_pad_mask=pad.to(cuda),
                            causal=causal),
             offset_buckets(places, places, edges, pad_mask=pad, query_pad_mask=pad, causal=causal))


@pytest.mark.parametrize("B,Nq,Nk", [(1, 1, 1), (2, 33, 130), (3, 181, 181), (1, 64, 128)])
def test_value_and_index_buckets(cuda, B, Nq, Nk):
    g = torch.Generator().manual_seed(B * Nq)
    values = torch.randn(B, Nq, Nk, generator=g) * 3.0
    values[0, 0, 0] = math.nan
    pad = torch.rand(B, Nk, generator=g) < 0.3
    edges = sorted({x for x in values.flatten()[:40].tolist() if x == x})[:39]  # (a NaN has no place in an order)
    for gradients in (True, False):
        same(value_buckets(values.to(cuda), edges, pad_mask=pad.to(cuda), cutoff=4.0, gradients=gradients),
             value_buckets(values, edges, pad_mask=pad, cutoff=4.0, gradients=gradients))
    index = torch.randint(-3, 70, (B, Nq, Nk), generator=g)
    index[0, 0, 0] = 2 ** 32 + 1
    for t in (index, index.int(), index.clamp_min(0).to(torch.uint8)):
        same(index_buckets(t.to(cuda), 30, query_pad_mask=torch.zeros(B, Nq, dtype=torch.int64, device=cuda)), index_buckets(t, 30))


def test_empty_calls(cuda):
    for B, N in ((0, 5), (2, 0)):
        b = distance_buckets(torch.zeros(B, N, 3, device=cuda), [1.0])
        assert b.index.shape == (B, N, N)
        table = torch.zeros(2, 3, device=cuda, requires_grad=True)
        bias = bucket_bias(table, b)
        assert bias.shape == (B, 3, N, N)
        bias.sum().backward()
        assert not table.grad.any()


DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Nq,Nk,K", [(1, 1, 1, 1, 1), (2, 8, 29, 29, 32), (3, 5, 64, 181, 64), (2, 12, 130, 257, 17),
                                         (1, 3, 1, 1000, 8), (1, 128, 7, 15, 5)])
def test_bias_and_its_gradient(cuda, B, H, Nq, Nk, K, dtype):
    g = torch.Generator(device=cuda).manual_seed(H * Nk)
    index = torch.randint(-1, K, (B, Nq, Nk), generator=g, device=cuda, dtype=torch.int32)
    buckets = index_buckets(index, K)
    for table_dtype in (dtype, torch.float32):
        table = torch.randn(K, H, generator=g, device=cuda).to(table_dtype).requires_grad_(True)
        bias = bucket_bias(table, buckets, dtype=dtype)
        want = dense(buckets.index, table.detach())
        assert bias.dtype == dtype and torch.equal(bias.double(), want.to(dtype).double())
        go = torch.randn(bias.shape, generator=g, device=cuda).to(dtype)
        go[0, :, :, 0] *= 1000.0
        go[(index < 0)[:, None].expand_as(go)] = math.nan  # pairs that are left out count for nothing
        (grad,) = torch.autograd.grad(bias, table, go)
        masked = torch.where((index >= 0)[:, None], go.double(), 0.0)
        for c in range(K):
            terms = torch.where((index == c)[:, None], masked, 0.0)
            exact, spread = terms.sum((0, 2, 3)), terms.abs().sum((0, 2, 3))
            # fp32 sums of at most 4096 terms a lane and of 256 lanes: a step each, on partial sums below the spread
            off = (grad[c].double() - exact).abs()
            assert (off <= spread * 4096 * 2.0 ** -24 + step(table_dtype) * exact.abs()).all()
        (again,) = torch.autograd.grad(bucket_bias(table, buckets, dtype=dtype), table, go)
        assert torch.equal(grad, again)


def test_bias_of_a_shared_batch(cuda):
    index = torch.randint(0, 6, (1, 40, 40), device=cuda)
    buckets = index_buckets(index, 6)
    table = torch.randn(6, 4, device=cuda, requires_grad=True)
    bias = bucket_bias(table, buckets, batch=3)
    assert torch.equal(bias, dense(buckets.index, table.detach()).float().expand(3, 4, 40, 40))
    go = torch.randn_like(bias)
    (grad,) = torch.autograd.grad(bias, table, go)
    for c in range(6):
        assert torch.allclose(grad[c].double(), torch.where((index == c)[:, None], go.double(), 0.0).sum((0, 2, 3)), atol=1e-3)
    # an upstream gradient that is itself a broadcast view
    (ones,) = torch.autograd.grad(bucket_bias(table, buckets, batch=3).sum(), table)
    assert torch.equal(ones, torch.stack([(index == c).sum().float().expand(4) * 3 for c in range(6)]))


def test_bias_of_more_than_2_31_entries(cuda):
    """(the index of one atom pair row is shared; 2.2e9 entries of bias)"""
    N, H = 4700, 100
    index = torch.randint(0, 8, (1, N, N), device=cuda, dtype=torch.int32)
    buckets = index_buckets(index, 8)
    table = torch.randn(8, H, device=cuda).bfloat16()
    bias = bucket_bias(table, buckets)
    assert bias.numel() > 2 ** 31
    for h, i in ((0, 0), (H - 1, N - 1), (H - 3, 17)):
        assert torch.equal(bias[0, h, i], table[:, h][index[0, i].long()])


def test_tables_with_infinities_and_lowest_values(cuda):
    index = torch.randint(0, 4, (1, 9, 30), device=cuda)
    for dtype in DTYPES:
        table = torch.tensor([[0.0], [-math.inf], [torch.finfo(dtype).min], [math.inf]], device=cuda, dtype=dtype)
        assert torch.equal(bucket_bias(table, index_buckets(index, 4))[0, 0], table[:, 0][index[0]])


def test_refused_bias(cuda):
    buckets = index_buckets(torch.zeros(1, 3, 3, dtype=torch.int32, device=cuda), 4)
    with pytest.raises(RuntimeError, match="only supports"):
        bucket_bias(torch.zeros(4, 2, dtype=torch.float64, device=cuda), buckets)
    with pytest.raises(RuntimeError, match="only supports"):
        bucket_bias(torch.zeros(4, 2, device=cuda), buckets, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="128 heads"):
        bucket_bias(torch.zeros(4, 129, device=cuda), buckets)
    with pytest.raises(RuntimeError, match="same device"):
        bucket_bias(torch.zeros(4, 2), buckets)


def test_buckets_and_bias_in_a_graph(cuda):
    coords = torch.randn(4, 70, 3, device=cuda)
    table = torch.randn(9, 8, device=cuda)
    edges = [0.3 * i for i in range(1, 9)]

    def step():
        b = distance_buckets(coords, edges)
        return bucket_bias(table, b), b.key_any

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        coords.copy_(torch.randn_like(coords))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_two_streams_at_once(cuda):
    index = [torch.randint(0, 16, (4, 300, 300), device=cuda) for _ in range(2)]
    table = torch.randn(16, 8, device=cuda, requires_grad=True)
    go = torch.randn(4, 8, 300, 300, device=cuda)
    want = [torch.autograd.grad(bucket_bias(table, index_buckets(i, 16)), table, go)[0] for i in index]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in index]
    got = []
    for s, i in zip(streams, index):
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(bucket_bias(table, index_buckets(i, 16)), table, go)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_distances_between_two_sets_through_the_c_entry(cuda):
    import ctypes

    from matterformer_amd import _native

    g = torch.Generator().manual_seed(11)
    B, Nq, Nk = 2, 70, 130
    a, b = torch.randn(B, Nq, 3, generator=g), torch.randn(1, Nk, 3, generator=g)
    edges = [0.5 * i for i in range(1, 8)]
    values = torch.full((B, Nq, Nk), 0, dtype=torch.uint8)
    d = a.double()[:, :, None] - b.double()[:, None]
    d2 = (d[..., 0] * d[..., 0] + d[..., 1] * d[..., 1]) + d[..., 2] * d[..., 2]
    for e in edges:
        values += d2 >= e * e
    values[d2 > 9.0] = MASKED
    at, bt = a.to(cuda), b.to(cuda)
    index = torch.zeros(B, Nq, 192, dtype=torch.uint8, device=cuda)
    index_t = torch.zeros(B, Nk, 128, dtype=torch.uint8, device=cuda)
    any_k, any_q = (torch.zeros(B, *s, dtype=torch.int64, device=cuda) for s in ((2, 3), (3, 2)))
    host = (ctypes.c_double * 7)(*edges)
    _native.launch("mf_pair_buckets", _native.MfPairBucketsArgs(
        query_pos=at.data_ptr(), key_pos=bt.data_ptr(), edges=ctypes.addressof(host), index=index.data_ptr(),
        index_t=index_t.data_ptr(), key_any=any_k.data_ptr(), query_any=any_q.data_ptr(), query_step=3 * Nq, key_step=0,
        cutoff=3.0, source=_native.MF_BUCKETS_DISTANCE, num_edges=7, buckets=8, batch=B, queries=Nq, keys=Nk), at.device)
    assert torch.equal(index[:, :, :Nk].cpu(), values) and index[:, :, Nk:].eq(MASKED).all()
    assert torch.equal(index_t[:, :, :Nq].cpu(), values.transpose(1, 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Nq,Nk", [(2, 3, 900, 3), (2, 2, 700, 15), (1, 3, 5000, 1), (2, 3, 301, 17), (1, 3, 3, 4099), (1, 2, 1, 9001),
                                       (3, 2, 13, 30), (2, 2, 200, 509)])
def test_planes_that_begin_anywhere(cuda, B, H, Nq, Nk, dtype):
    """Rows shorter than an access, longer than what a workgroup takes at once, and planes off 16 bytes."""
    test_bias_and_its_gradient(cuda, B, H, Nq, Nk, 23, dtype)


def test_a_gradient_off_16_bytes(cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    index = torch.randint(-1, 9, (2, 31, 33), generator=g, device=cuda, dtype=torch.int32)
    table = torch.randn(9, 5, generator=g, device=cuda).requires_grad_(True)
    bias = bucket_bias(table, index_buckets(index, 9))
    go = torch.randn(bias.numel() + 1, generator=g, device=cuda)[1:].view(bias.shape)
    assert go.data_ptr() % 16 and go.is_contiguous()
    (grad,) = torch.autograd.grad(bias, table, go, retain_graph=True)
    (same,) = torch.autograd.grad(bias, table, go.clone())
    assert torch.equal(grad, same)


# edges within 1024 steps of fp32 of each other: one, neighbours, of either sign, at zero and at the ends of the range
CLOSE_OFFSETS = [[1], [3], [64], [-64], [-3, -2], [-1, 0, 1], [5, 6, 7], [1000000, 1000001, 1000002],
                 [-1000002, -1000001, -1000000], [2 ** 40], [-(2 ** 53)], [2 ** 53 - 1, 2 ** 53]]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("edges", CLOSE_OFFSETS, ids=str)
def test_offsets_of_both_signs_about_close_edges(cuda, edges, causal):
    """Whole tiles of one bucket on either side of the diagonal, near places in no order, and places far apart."""
    g = torch.Generator().manual_seed(abs(edges[0]) % 1000)
    in_order = torch.arange(200)
    near = torch.randint(-100, 100, (2, 150), generator=g)
    far = torch.tensor([0, 2, 5, -7, 10 ** 6, 10 ** 6 + 1, -(10 ** 6), 2 ** 31, -(2 ** 31), 2 ** 40, -(2 ** 40), 2 ** 53, -(2 ** 53),
                        2 ** 61, -(2 ** 61)])
    for p in (in_order, near, far):
        same(offset_buckets(p.to(cuda), p.to(cuda), edges, causal=causal), offset_buckets(p, p, edges, causal=causal))
    one = torch.tensor([100])
    same(offset_buckets(one.to(cuda), in_order.to(cuda), edges, causal=causal, gradients=False),
         offset_buckets(one, in_order, edges, causal=causal, gradients=False))


def close_values():
    ends = [1e-45, 1e-38, 1.0, 3.5, 1e20, torch.finfo(torch.float32).max]
    single = [[s * e] for e in ends for s in (1.0, -1.0)] + [[0.0], [-0.0]]
    up = lambda x: torch.nextafter(torch.tensor(x), torch.tensor(math.inf)).item()
    return single + [[x, up(x), up(up(x))] for x in (1.0, -1.0, 1000.0, -1000.0, 0.0, -1e-45)]


@pytest.mark.parametrize("edges", close_values(), ids=str)
def test_values_of_both_signs_about_close_edges(cuda, edges):
    g = torch.Generator().manual_seed(3)
    values = torch.randn(2, 70, 90, generator=g) * torch.tensor([1.0, 1e4])[:, None, None]
    special = [0.0, -0.0, 1e-45, -1e-45, 1e-38, -1e-38, math.inf, -math.inf, math.nan, 3.4e38, -3.4e38, *edges,
               *(-e for e in edges)]
    values[0, 0, :len(special)] = torch.tensor(special)
    for cutoff in (None, 2.0):
        got = value_buckets(values.to(cuda), edges, cutoff=cutoff)
        same(got, value_buckets(values, edges, cutoff=cutoff))
    assert got.index[0, 0, special.index(math.inf)] == MASKED and got.index[0, 0, 8] == 0  # above the cutoff; a NaN


def test_a_bias_about_one_edge(cuda):
    """What the buckets are read for: keys before the query have the first entry, those behind it the second."""
    places = torch.arange(150, device=cuda)
    table = torch.tensor([[1.0], [2.0]], device=cuda)
    bias = bucket_bias(table, offset_buckets(places, places, [1]))[0, 0]
    assert torch.equal(bias, 1.0 + (places[None] > places[:, None]).float())


def test_more_tiles_than_one_launch(cuda):
    """(2^23 workgroups a launch; a tile an entry here)"""
    B = 2 ** 23 + 77
    g = torch.Generator(device=cuda).manual_seed(4)
    index = torch.randint(-1, 9, (B, 1, 1), generator=g, device=cuda, dtype=torch.int32)
    got = index_buckets(index, 9)
    want = torch.where(index < 0, MASKED, index)
    assert torch.equal(got.index.int(), want) and torch.equal(got.index_t.int(), want)
    assert torch.equal(got.key_any, (index >= 0).long()) and torch.equal(got.query_any, (index >= 0).long())
