"""Bucket blocks of the trunk on the GPU: against the same modules in 64 bits, packed and padded, in training, in a graph."""

import copy

import pytest
import torch

from matterformer_amd import _native
from matterformer_amd.bucket_attention import bucket_attention
from matterformer_amd.geometry import NonPeriodicGeometryAdapter, PeriodicGeometryAdapter
from matterformer_amd.geometry_bias import BucketedGeometryBias
from matterformer_amd.pair_buckets import distance_buckets, value_buckets
from matterformer_amd.token_packing import TokenPacking
from matterformer_amd.trunk import AdaLNBlock, AlternatingTrunk, BucketAttention

pytestmark = pytest.mark.gpu

EDGES = [0.4 * i for i in range(1, 24)]


def off(got, want):
    """Error relative to the norm."""
    got, want = got.detach().double(), want.detach().double().to(got.device)
    return float((got - want).norm() / want.norm())


def make_attn(cuda, d_model, heads, dtype):
    torch.manual_seed(d_model + heads)
    attn = BucketAttention(d_model, heads, len(EDGES) + 1)
    torch.nn.init.normal_(attn.bias_table)
    torch.nn.init.normal_(attn.attn.in_proj_bias, std=0.1)
    return attn.to(cuda, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d_model,heads", [(256, 8), (384, 8), (128, 1)])
def test_attention_module(cuda, d_model, heads, dtype):
    attn = make_attn(cuda, d_model, heads, dtype)
    exact = copy.deepcopy(attn).double()
    exact.impl = "torch"
    h = torch.randn(3, 70, d_model, device=cuda).to(dtype)
    pad = torch.arange(70, device=cuda)[None] >= torch.tensor([[70], [41], [3]], device=cuda)
    buckets = distance_buckets(torch.randn(3, 70, 3, device=cuda) * 3.0, EDGES, pad_mask=pad, cutoff=12.0)
    x, y = h.clone().requires_grad_(True), h.double().requires_grad_(True)
    got, want = attn(x, buckets), exact(y, buckets)
    assert attn._last_impl_used == "triton" and exact._last_impl_used == "torch"
    # a chain of at most eight roundings to the type, each half a step of what it rounds
    u = torch.finfo(dtype).eps / 2
    assert off(got, want) <= 8 * u
    go = torch.randn_like(got)
    grads = torch.autograd.grad(got, [x, *attn.parameters()], go)
    exacts = torch.autograd.grad(want, [y, *exact.parameters()], go.double())
    for (name, _), a, b in zip([("h", None), *attn.named_parameters()], grads, exacts):
        assert off(a, b) <= 16 * u, name  # forward and backward
    with torch.no_grad():
        assert torch.equal(attn(h, buckets), got)


def test_fp32_modules(cuda):
    """Inference runs the core in bfloat16; training takes the torch path, autocast the kernels."""
    attn = make_attn(cuda, 128, 2, torch.float32)
    h = torch.randn(2, 50, 128, device=cuda)
    buckets = distance_buckets(torch.randn(2, 50, 3, device=cuda), EDGES)
    out = attn(h, buckets)
    assert attn._last_impl_used == "torch"
    with torch.no_grad():
        assert off(attn(h, buckets), out) <= 8 * 2.0 ** -9 and attn._last_impl_used == "triton"
    with torch.autocast("cuda", dtype=torch.bfloat16):
        trained = attn(h, buckets)
        assert attn._last_impl_used == "triton"
    trained.float().square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in attn.parameters())
    attn.attn.dropout = 0.5
    attn.train()(h, buckets)
    assert attn._last_impl_used == "torch"
    attn.impl = "triton"
    with pytest.raises(RuntimeError, match="dropout"):
        attn(h, buckets)


def make_trunk(cuda, dtype, **kw):
    torch.manual_seed(5)
    trunk = AlternatingTrunk(256, 4, 3, schedule=["bucket", "simplicial", "bucket"], bucket_edges=EDGES, **kw)
    for block in trunk.blocks:
        torch.nn.init.normal_(block.ada_ln[-1].weight, std=0.05)
        if block.attn_type == "bucket":
            torch.nn.init.normal_(block.attn.bias_table)
    return trunk.to(cuda, dtype)


def batch(cuda, dtype, B=4, N=90):
    g = torch.Generator(device=cuda).manual_seed(7)
    x = torch.randn(B, N, 256, generator=g, device=cuda).to(dtype)
    cond = torch.randn(B, 256, generator=g, device=cuda).to(dtype)
    coords = torch.randn(B, N, 3, generator=g, device=cuda) * 2.0
    pad = torch.arange(N, device=cuda)[None] >= torch.randint(20, N, (B, 1), generator=g, device=cuda)
    return x, cond, coords, pad


def test_trunk_packed_and_padded(cuda):
    trunk = make_trunk(cuda, torch.bfloat16).eval()
    x, cond, coords, pad = batch(cuda, torch.bfloat16)
    with torch.no_grad():
        packed = trunk(x, cond, coords, pad)
        trunk.pack_tokens = False
        padded = trunk(x, cond, coords, pad)
        for block in trunk.blocks:  # the same trunk in 64 bits
            block.attn.impl = "torch"
        exact = trunk.double()(x.double(), cond.double(), coords, pad)
    assert not packed[pad].any() and not padded[pad].any()
    # three blocks of about ten roundings each
    assert off(packed, exact) <= 30 * 2.0 ** -9 and off(padded, exact) <= 30 * 2.0 ** -9


def test_trunk_trains(cuda):
    """One step of everything together: buckets, their bias as simplicial terms, attention, gradients of all tables."""
    bias = BucketedGeometryBias(4, EDGES)
    for p in (bias.u_table, bias.v_table, bias.w_table):
        torch.nn.init.normal_(p, std=0.3)
    trunk = make_trunk(cuda, torch.bfloat16, geometry_adapter=NonPeriodicGeometryAdapter(), simplicial_geometry_bias=bias)
    x, cond, coords, pad = batch(cuda, torch.bfloat16, N=60)
    sigma = torch.tensor([0.5, 1.0, 2.0, 3.0], device=cuda)
    exact = copy.deepcopy(trunk).cpu().double()
    out = trunk(x, cond, coords, pad, sigma=sigma)
    want = exact(x.cpu().double(), cond.cpu().double(), coords.cpu(), pad.cpu(), sigma=sigma.cpu())
    assert all(b.attn._last_impl_used == "triton" for b in trunk.blocks if b.attn_type == "bucket")
    go = torch.randn_like(out)
    out.backward(go)
    want.backward(go.cpu().double())
    assert off(out, want) <= 30 * 2.0 ** -9
    for (name, p), e in zip(trunk.named_parameters(), exact.parameters()):
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        if e.grad.norm() > 0 and "table" in name:
            assert off(p.grad, e.grad) <= 60 * 2.0 ** -9, name


def test_periodic_geometry(cuda):
    """Minimum-image distances through the adapter's pair_dist: the bias on the GPU is that on the CPU."""
    adapter, bias = PeriodicGeometryAdapter(), BucketedGeometryBias(4, EDGES, use_noise_gate=False)
    torch.nn.init.normal_(bias.u_table)
    frac, lattice = torch.rand(2, 30, 3), torch.tensor([[1.5, 1.6, 1.4, 0.1, 0.0, -0.1]] * 2)
    geom = adapter.to(cuda)(coords=frac.to(cuda), lattice=lattice.to(cuda))
    on_cpu = type(geom)(**{k: v.cpu() if torch.is_tensor(v) else v for k, v in vars(geom).items()})
    want = bias.build_structured_bias_inputs(on_cpu, 30)[0]
    got = bias.to(cuda).build_structured_bias_inputs(geom, 30)[0]
    assert torch.equal(got.u.cpu(), want.u)


def test_trunk_in_a_graph(cuda):
    trunk = make_trunk(cuda, torch.bfloat16).eval()
    x, cond, coords, pad = batch(cuda, torch.bfloat16)
    packing = TokenPacking(pad)
    with torch.no_grad():
        trunk(x, cond, coords, pad, packing=packing)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = trunk(x, cond, coords, pad, packing=packing)
        for _ in range(3):
            x.copy_(torch.randn_like(x))
            coords.copy_(torch.randn_like(coords) * 2.0)
            want = trunk(x, cond, coords, pad, packing=packing)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want)


def test_periodic_trunk(cuda):
    """Bucket blocks on periodic cells: padded and packed forwards and a step of training against the same trunk in 64 bits,
    whose buckets are those of the same distances."""
    adapter = PeriodicGeometryAdapter()
    trunk = make_trunk(cuda, torch.bfloat16, geometry_adapter=adapter, bucket_cutoff=4.0)
    x, cond, _, pad = batch(cuda, torch.bfloat16)
    g = torch.Generator(device=cuda).manual_seed(8)
    frac = torch.rand(*x.shape[:2], 3, generator=g, device=cuda)
    lattice = torch.tensor([[1.5, 1.6, 1.4, 0.1, 0.0, -0.1], [1.1, 1.2, 1.0, 0.0, 0.2, 0.1]] * 2, device=cuda)
    exact = copy.deepcopy(trunk).double()
    for block in exact.blocks:
        block.attn.impl = "torch"
    seen = []
    exact.blocks[0].attn.register_forward_pre_hook(lambda module, args: seen.append(args[1].index))
    want = exact(x.double(), cond.double(), frac, pad, lattice=lattice)
    dist = adapter(coords=frac, pad_mask=pad, lattice=lattice).pair_dist
    counts = torch.stack([dist >= torch.tensor(e, device=cuda) for e in EDGES]).sum(0)
    left_out = pad[:, None, :] | pad[:, :, None] | (dist > 4.0)
    assert torch.equal(seen[0].long(), torch.where(left_out, 64, counts))
    out = trunk(x, cond, frac, pad, lattice=lattice)
    assert all(b.attn._last_impl_used == "triton" for b in trunk.blocks if b.attn_type == "bucket")
    assert off(out, want) <= 30 * 2.0 ** -9
    go = torch.randn_like(out)
    out.backward(go)
    want.backward(go.double())
    for block, other in zip(trunk.blocks, exact.blocks):
        if block.attn_type == "bucket":
            assert off(block.attn.bias_table.grad, other.attn.bias_table.grad) <= 60 * 2.0 ** -9
    with torch.no_grad():
        packed = trunk.eval()(x, cond, frac, pad, lattice=lattice)
        trunk.pack_tokens = False
        padded = trunk(x, cond, frac, pad, lattice=lattice)
    assert off(packed, want) <= 30 * 2.0 ** -9 and off(padded, want) <= 30 * 2.0 ** -9


def test_periodic_trunk_in_a_graph(cuda):
    trunk = make_trunk(cuda, torch.bfloat16, geometry_adapter=PeriodicGeometryAdapter()).eval()
    x, cond, _, pad = batch(cuda, torch.bfloat16)
    frac = torch.rand(*x.shape[:2], 3, device=cuda)
    lattice = torch.tensor([[1.5, 1.6, 1.4, 0.1, 0.0, -0.1]] * 4, device=cuda)
    packing = TokenPacking(pad)
    with torch.no_grad():
        trunk(x, cond, frac, pad, lattice=lattice, packing=packing)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = trunk(x, cond, frac, pad, lattice=lattice, packing=packing)
        for _ in range(3):
            x.copy_(torch.randn_like(x))
            frac.copy_(torch.rand_like(frac))
            want = trunk(x, cond, frac, pad, lattice=lattice, packing=packing)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want)


class OlderBlock(AdaLNBlock):
    """A block whose packed methods know the local and simplicial inputs only."""

    def forward_packed(self, xp, cond_emb, packing, *, knn_mask=None, terms=None):
        return super().forward_packed(xp, cond_emb, packing, knn_mask=knn_mask, terms=terms)

    def _attention_packed(self, h, packing, knn_mask, terms):
        return super()._attention_packed(h, packing, knn_mask, terms)


@pytest.mark.parametrize("adaln", [True, False])
def test_packed_blocks_without_a_place_for_buckets(cuda, adaln):
    torch.manual_seed(5)
    trunk = AlternatingTrunk(256, 4, 3, schedule=["bucket", "simplicial", "knn_local"], bucket_edges=EDGES, knn_k=8,
                             use_adaln_conditioning=adaln).to(cuda, torch.bfloat16).eval()
    x, cond, coords, pad = batch(cuda, torch.bfloat16)
    with torch.no_grad():
        want = trunk(x, cond, coords, pad)
        assert all(b.attn._last_impl_used == "triton" for b in trunk.blocks)
        for block in trunk.blocks[1:]:
            block.__class__ = OlderBlock
        assert torch.equal(trunk(x, cond, coords, pad), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("periodic", [False, True])
def test_a_torch_trunk_runs_no_bucket_kernel(cuda, periodic, dtype, monkeypatch):
    """impl="torch" is the torch formulation throughout, the buckets too; they are those that the kernel gives."""
    trunk = make_trunk(cuda, dtype, bucket_impl="torch", simplicial_impl="torch", bucket_cutoff=6.0,
                       geometry_adapter=PeriodicGeometryAdapter() if periodic else NonPeriodicGeometryAdapter())
    x, cond, coords, pad = batch(cuda, dtype)
    lattice = torch.tensor([[1.5, 1.6, 1.4, 0.1, 0.0, -0.1]] * 4, device=cuda) if periodic else None
    launch = _native.launch

    def only_geometry(name, *args):
        assert "bucket" not in name
        launch(name, *args)

    seen = []
    trunk.blocks[0].attn.register_forward_pre_hook(lambda module, args: seen.append(args[1]))
    monkeypatch.setattr(_native, "launch", only_geometry)
    out = trunk(x, cond, coords, pad, lattice=lattice)
    out.square().sum().backward()
    assert all(b.attn._last_impl_used == "torch" for b in trunk.blocks)
    assert trunk.blocks[0].attn.bias_table.grad.abs().max() > 0
    monkeypatch.undo()
    if periodic:
        dist = trunk.geometry_adapter(coords=coords, pad_mask=pad, lattice=lattice).pair_dist
        want = value_buckets(dist, EDGES, pad_mask=pad, query_pad_mask=pad, cutoff=6.0)
    else:
        want = distance_buckets(coords, EDGES, pad_mask=pad, cutoff=6.0)
    assert torch.equal(seen[0].index, want.index) and torch.equal(seen[0].index_t, want.index_t)
    # the kernels, which read another layout, refuse such buckets
    q = torch.zeros(4, 2, 90, 32, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="distance_buckets"):
        bucket_attention(q, q, q, torch.zeros(len(EDGES) + 1, 2, device=cuda), seen[0])


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("table", [torch.float64, torch.float32])
def test_float64_modules_take_the_torch_path(cuda, table, autocast):
    """In inference and in training, autocast or not (which leaves 64-bit operands alone): no core in 16 bits."""
    attn = make_attn(cuda, 128, 2, torch.float64)
    attn.bias_table.data = attn.bias_table.data.to(table)
    h = torch.randn(2, 50, 128, device=cuda).double()
    coords = torch.randn(2, 50, 3, device=cuda)
    buckets = distance_buckets(coords, EDGES)
    other = copy.deepcopy(attn).cpu()
    want = other(h.cpu(), distance_buckets(coords.cpu(), EDGES))
    for grad in (False, True):
        with torch.set_grad_enabled(grad), torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            out = attn(h, buckets)
        assert attn._last_impl_used == "torch" and out.dtype == torch.float64
        # sums of at most 128 fp64 terms, some products deep
        assert off(out, want) <= 2.0 ** -40
    out.sum().backward()
    assert all(p.grad.dtype == p.dtype for p in attn.parameters())
    attn.impl = "triton"
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="bucket attention needs"):
            attn(h, buckets)


def test_whole_types_of_indexes(cuda):
    from matterformer_amd.pair_buckets import index_buckets

    for dtype in (torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64, torch.uint64):
        top = torch.iinfo(dtype).max
        numbers = [n for n in (0, 3, 4, 63, 64, 255, 2 ** 31, 2 ** 32, 2 ** 63, top) if n <= top]
        index = torch.tensor(numbers, dtype=dtype).view(1, 1, -1)
        assert index_buckets(index.to(cuda), 4).index.flatten().tolist() == [n if n < 4 else 64 for n in numbers]
