"""Pair buckets, their bias and the attention with it on the CPU: the torch formulations against loops, refusals, and the C
entries' checks and structs."""

import ctypes
import math
import re
import shutil
import subprocess

import pytest
import torch

from matterformer_amd import _native
from matterformer_amd.bucket_attention import bucket_attention, bucket_attention_torch
from matterformer_amd.pair_buckets import (MASKED, PairBuckets, bucket_bias, check_layout, distance_buckets, index_buckets,
                                           offset_buckets, offset_edges, value_buckets)
from tests.bucket_reference import attention
from tests.test_capi import HEADER


def test_distance_buckets_count_edges():
    g = torch.Generator().manual_seed(3)
    coords = torch.randn(2, 9, 3, generator=g)
    pad = torch.zeros(2, 9, dtype=torch.bool)
    pad[1, 6:] = True
    edges = [0.5, 1.0, 1.5, 2.5]
    b = distance_buckets(coords, edges, pad_mask=pad, cutoff=3.0)
    assert b.num_buckets == 5 and (b.batch, b.queries, b.keys) == (2, 9, 9)
    for n in range(2):
        for i in range(9):
            for j in range(9):
                d = math.dist(coords[n, i].tolist(), coords[n, j].tolist())
                want = MASKED if d > 3.0 or pad[n, i] or pad[n, j] else sum(d >= e for e in edges)
                assert b.index[n, i, j] == want
    assert torch.equal(b.index_t, b.index.transpose(1, 2))
    assert torch.equal(b.allowed(), b.index != MASKED)


def test_a_distance_at_an_edge_is_on_its_exact_side():
    # 3-4-5: at the edge; a step of fp32 to either side of it is below or above
    x = torch.tensor([[[0.0, 0, 0], [3.0, 4.0, 0.0], [3.0, math.nextafter(4.0, 0.0), 0.0]]])
    x[0, 2, 1] = torch.nextafter(torch.tensor(4.0), torch.tensor(0.0))
    b = distance_buckets(x, [5.0])
    assert b.index[0, 0].tolist() == [0, 1, 0]
    assert distance_buckets(x, [6.0], cutoff=5.0).index[0, 0].tolist() == [0, 0, 0]
    assert distance_buckets(x, [6.0], cutoff=math.nextafter(5.0, 0) - 1e-6).index[0, 0].tolist()[1] == MASKED


def test_offset_value_and_index_buckets():
    places = torch.tensor([5, 6, 9, 200])
    b = offset_buckets(places, places, [-3, 0, 1, 4])
    for i, p in enumerate(places.tolist()):
        for j, r in enumerate(places.tolist()):
            assert b.index[0, i, j] == sum(r - p >= e for e in (-3, 0, 1, 4))
    causal = offset_buckets(places[1:2], places, [0], causal=True, gradients=False)
    assert causal.index.tolist() == [[[0, 1, MASKED, MASKED]]] and causal.index_t is None
    both = offset_buckets(places[None], places.int(), [0], pad_mask=torch.tensor([[False, False, True, False]] * 3),
                          query_pad_mask=torch.tensor([[False] * 4, [True] * 4, [False] * 4]))
    assert both.batch == 3 and both.index[1].eq(MASKED).all() and both.index[0, :, 2].eq(MASKED).all()
    v = value_buckets(torch.tensor([[[0.0, 1.0, math.nan], [2.0, math.inf, -1.0]]]), [1.0, 2.0], cutoff=2.5)
    assert v.index.tolist() == [[[0, 1, 0], [2, MASKED, 0]]]
    i = index_buckets(torch.tensor([[[0, 3, 4, -1, 2 ** 32 + 1]]]), 4)
    assert i.index.tolist() == [[[0, 3, MASKED, MASKED, MASKED]]]


@pytest.mark.parametrize("buckets", [1, 2, 3, 8, 31, 32, 64])
@pytest.mark.parametrize("causal", [False, True])
def test_offset_edges(buckets, causal):
    edges = offset_edges(buckets, 1000, causal=causal)
    assert len(edges) == buckets - 1 and all(a < b for a, b in zip(edges, edges[1:]))
    assert not causal or all(e <= 0 for e in edges)
    assert all(abs(e) <= 1000 for e in edges)
    if buckets >= 8:  # near zero every offset has a bucket of its own
        near = offset_buckets(torch.tensor([0]), torch.tensor([-2, -1, 0]), edges).index[0, 0].tolist()
        assert near == sorted(set(near))


def test_bias_and_attention_follow_the_formulas():
    g = torch.Generator().manual_seed(5)
    index = torch.randint(-1, 6, (2, 5, 7), generator=g)
    buckets = index_buckets(index, 6)
    table = torch.randn(6, 4, generator=g, dtype=torch.float64)
    bias = bucket_bias(table.float(), buckets)
    for b in range(2):
        for i in range(5):
            for j in range(7):
                c = int(index[b, i, j])
                want = table[c].float() if c >= 0 else torch.full((4,), -math.inf)
                assert torch.equal(bias[b, :, i, j], want)
    q, go = (torch.randn(2, 4, 5, 8, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(2, 2, 7, 8, generator=g, dtype=torch.float64) for _ in range(2))
    index[0, 3] = -1
    buckets = index_buckets(index, 6)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, table)]
    out, lse = bucket_attention(*leaves, buckets, scale=0.3, return_lse=True)
    grads = torch.autograd.grad(out, leaves, go)
    r, _ = attention(q, k, v, table, buckets.index, 0.3, go)
    for got, name in zip((out, lse.double(), *grads), ("out", "lse", "dq", "dk", "dv", "dtable")):
        assert torch.allclose(got, r[name], rtol=1e-6, atol=1e-6 if name == "lse" else 1e-12), name
    assert not out[0, :, 3].any() and not lse[0, :, 3].any()


def test_rows_without_a_pair_may_hold_anything():
    torch.manual_seed(11)
    pad = torch.tensor([[False] * 5, [False, False, True, True, True]])
    buckets = distance_buckets(torch.randn(2, 5, 3), [0.5, 1.0, 2.0], pad_mask=pad)
    clean = [torch.randn(2, 4, 5, 8, dtype=torch.float64), torch.randn(2, 2, 5, 8, dtype=torch.float64),
             torch.randn(2, 2, 5, 8, dtype=torch.float64)]
    table, go = torch.randn(4, 4, dtype=torch.float64), torch.randn(2, 4, 5, 8, dtype=torch.float64)
    results = []
    for fill in (0.0, math.nan, math.inf):
        q, k, v, g = (t.masked_fill(pad[:, None, :, None], fill) for t in (*clean, go))
        leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
        out, lse = bucket_attention(*leaves, buckets, return_lse=True)
        out.backward(g)
        results.append([out.detach(), lse.detach(), *(t.grad for t in leaves)])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


def test_refusals():
    c = torch.zeros(1, 4, 3)
    for edges in ([1.0, 1.0], [2.0, 1.0], [math.nan], [math.inf], [1e39], list(range(1, 65)), [-1.0, 2.0]):
        with pytest.raises(ValueError):
            distance_buckets(c, edges)
    with pytest.raises(ValueError, match="coords"):
        distance_buckets(torch.zeros(1, 4, 2), [1.0])
    for cutoff in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="cutoff"):
            distance_buckets(c, [1.0], cutoff=cutoff)
    with pytest.raises(ValueError, match="pad_mask"):
        distance_buckets(c, [1.0], pad_mask=torch.zeros(1, 5, dtype=torch.bool))
    p = torch.arange(4)
    with pytest.raises(ValueError, match="whole"):
        offset_buckets(p, p, [0.5])
    with pytest.raises(ValueError, match="2\\^53"):
        offset_buckets(p, p, [2 ** 53 + 2])
    with pytest.raises(RuntimeError, match="whole"):
        offset_buckets(p.float(), p, [0])
    with pytest.raises(ValueError, match="rows"):
        offset_buckets(torch.zeros(2, 4, dtype=torch.long), torch.zeros(3, 4, dtype=torch.long), [0])
    for n in (0, 65):
        with pytest.raises(ValueError, match="num_buckets"):
            index_buckets(torch.zeros(1, 1, 1, dtype=torch.int32), n)
        with pytest.raises(ValueError, match="num_buckets"):
            offset_edges(n, 100)
    with pytest.raises(ValueError, match="max_offset"):
        offset_edges(64, 10)
    b = index_buckets(torch.zeros(2, 3, 5, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="table"):
        bucket_bias(torch.zeros(5, 2), b)
    with pytest.raises(TypeError, match="PairBuckets"):
        bucket_bias(torch.zeros(4, 2), b.index)
    with pytest.raises(ValueError, match="batch"):
        bucket_bias(torch.zeros(4, 2), b, batch=3)
    q, k = torch.zeros(2, 4, 3, 8), torch.zeros(2, 2, 5, 8)
    table = torch.zeros(4, 4)
    for args, match in (((q[0], k, k, table, b), "shape"), ((q, k[:1], k[:1], table, b), "shape"),
                        ((q, k[..., :4], k[..., :4], table, b), "shape"), ((q, k, k[:, :1], table, b), "shape"),
                        ((q[:, :3], k, k, table[:, :3], b), "divide"), ((q, k, k, table[:, :3], b), "table"),
                        ((q[:, :, :2], k, k, table, b), "buckets must be of"),
                        ((q.repeat(2, 1, 1, 1), k.repeat(2, 1, 1, 1), k.repeat(2, 1, 1, 1), table, b), "buckets must be of")):
        with pytest.raises(ValueError, match=match):
            bucket_attention(*args)
    with pytest.raises(ValueError, match="finite"):
        bucket_attention(q, k, k, table, b, scale=math.inf)


def test_layout_of_foreign_buckets_is_refused():
    def rows(*shape):
        return torch.zeros(*shape[:2], (shape[2] + 63) // 64 * 64, dtype=torch.uint8)[:, :, :shape[2]]

    def make(**kw):
        t = dict(index=rows(2, 70, 5), index_t=rows(2, 5, 70), num_buckets=4,
                 key_any=torch.zeros(2, 2, 1, dtype=torch.int64), query_any=torch.zeros(2, 1, 2, dtype=torch.int64))
        t.update(kw)
        return PairBuckets(**t)

    check_layout(make())
    check_layout(make(index_t=None))
    for kw in (dict(index=rows(2, 70, 5).contiguous()), dict(index=rows(2, 70, 5).int()), dict(index_t=rows(2, 5, 71)),
               dict(key_any=None), dict(query_any=torch.zeros(2, 2, 1, dtype=torch.int64)),
               dict(key_any=torch.zeros(2, 2, 1)), dict(key_any=torch.zeros(2, 1, 2, dtype=torch.int64).transpose(1, 2)[:1])):
        with pytest.raises(ValueError, match="distance_buckets"):
            check_layout(make(**kw))


def test_structs_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = {"mf_pair_buckets_args": _native.MfPairBucketsArgs, "mf_bucket_bias_args": _native.MfBucketBiasArgs,
               "mf_bucket_attn_args": _native.MfBucketAttnArgs, "mf_bucket_attn_bwd_args": _native.MfBucketAttnBwdArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mf_capi.h"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        member = lambda f: re.sub(r"^(.*_stride)(\d)$", r"\1[\2]", f)  # an array's elements are fields of their own
        lines += [f'  printf("%zu\\n", offsetof({name}, {member(f[0])}));' for f in py._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run([cc, f"-I{HEADER.parent}", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    want = []
    for py in structs.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f[0]).offset for f in py._fields_]
    assert [int(x) for x in got] == want


FAKE = 1 << 20  # never dereferenced: every call below fails validation first
INVALID, UNSUPPORTED = _native.MF_ERR_INVALID_ARGUMENT, _native.MF_ERR_UNSUPPORTED


def refused(fn, args, status, match):
    assert fn(args, None) == status
    assert match in _native.last_error(), _native.last_error()


def test_buckets_entry_refuses_before_any_device_call():
    lib = _native.lib()
    edges = (ctypes.c_double * 3)(1.0, 2.0, 3.0)

    def args(edge=edges, **kw):
        a = dict(query_pos=FAKE, key_pos=FAKE, edges=ctypes.addressof(edge), index=FAKE, index_t=FAKE, key_any=FAKE,
                 query_any=FAKE, cutoff=-1.0, source=0, num_edges=3, buckets=4, batch=1, queries=5, keys=5)
        a.update(kw)
        return _native.MfPairBucketsArgs(**a)

    refused(lib.mf_pair_buckets, None, INVALID, "args is NULL")
    for kw, status, match in ((dict(source=4), INVALID, "source"), (dict(query_pos=None), INVALID, "non-NULL"),
                              (dict(source=2), INVALID, "non-NULL"), (dict(index=None), INVALID, "non-NULL"),
                              (dict(query_any=None), INVALID, "non-NULL"), (dict(batch=-1), INVALID, "non-negative"),
                              (dict(source=1), INVALID, "one set"), (dict(keys=6), INVALID, "one set"),
                              (dict(index_t=FAKE + 16), INVALID, "one set"), (dict(buckets=65), UNSUPPORTED, "[1, 64]"),
                              (dict(num_edges=2), INVALID, "buckets - 1"), (dict(cutoff=math.nan), INVALID, "NaN"),
                              (dict(queries=2 ** 24 + 1, keys=2 ** 24 + 1), UNSUPPORTED, "2^24"),
                              (dict(index=FAKE + 8, index_t=FAKE + 8), INVALID, "aligned")):
        refused(lib.mf_pair_buckets, args(**kw), status, match)
    for edge in ((1.0, 1.0, 2.0), (1.0, math.nan, 2.0), (-1.0, 0.0, 1.0), (0.0, 1.0, 1e300)):
        host = (ctypes.c_double * 3)(*edge)
        refused(lib.mf_pair_buckets, args(edge=host), INVALID, "edges")
    assert lib.mf_pair_buckets(args(batch=0), None) == _native.MF_OK


def test_more_tiles_than_32_bits_count_are_refused():
    args = _native.MfPairBucketsArgs(values=FAKE, index=FAKE, index_t=2 * FAKE, key_any=3 * FAKE, query_any=4 * FAKE,
                                     source=_native.MF_BUCKETS_INDEX, buckets=4, batch=2 ** 30, queries=65, keys=65)
    refused(_native.lib().mf_pair_buckets, args, UNSUPPORTED, "too large")
    args.batch, args.queries, args.keys = 1, 2 ** 24, 2 ** 24
    refused(_native.lib().mf_pair_buckets, args, UNSUPPORTED, "too large")


def test_bias_entries_refuse_before_any_device_call():
    lib = _native.lib()

    def args(**kw):
        a = dict(index=FAKE, table=FAKE, bias=FAKE, dtable=FAKE, index_batch=2, batch=2, heads=3, queries=4, keys=5, buckets=6,
                 table_dtype=0, bias_dtype=2)
        a.update(kw)
        return _native.MfBucketBiasArgs(**a)

    for fn in (lib.mf_bucket_bias, lib.mf_bucket_bias_bwd):
        refused(fn, None, INVALID, "args is NULL")
        for kw, status, match in ((dict(index=None), INVALID, "non-NULL"), (dict(bias=None), INVALID, "non-NULL"),
                                  (dict(keys=-1), INVALID, "non-negative"), (dict(index_batch=3), INVALID, "index_batch"),
                                  (dict(buckets=0), UNSUPPORTED, "[1, 64]"), (dict(heads=129), UNSUPPORTED, "128"),
                                  (dict(queries=2 ** 24 + 1), UNSUPPORTED, "2^24"), (dict(bias_dtype=3), UNSUPPORTED, "float32"),
                                  (dict(index=FAKE + 1), INVALID, "aligned"), (dict(bias=FAKE + 2), INVALID, "aligned")):
            refused(fn, args(**kw), status, match)
    refused(lib.mf_bucket_bias, args(table=None), INVALID, "non-NULL")
    refused(lib.mf_bucket_bias_bwd, args(dtable=None), INVALID, "non-NULL")
    refused(lib.mf_bucket_bias_bwd, args(), INVALID, "workspace")
    need = lib.mf_bucket_bias_bwd_workspace_size(args())
    refused(lib.mf_bucket_bias_bwd, args(workspace=FAKE, workspace_bytes=need - 1), INVALID, "workspace")
    for fn in (lib.mf_bucket_bias, lib.mf_bucket_bias_bwd):
        refused(fn, args(batch=2 ** 20, index_batch=1, queries=2 ** 13, keys=2 ** 10), UNSUPPORTED, "too large")
    assert lib.mf_bucket_bias(args(heads=0), None) == _native.MF_OK
    assert lib.mf_bucket_bias_bwd_workspace_size(args(queries=0)) == 0


ATTN = dict(q=FAKE, k=FAKE, v=FAKE, table=FAKE, index=FAKE, key_any=FAKE, query_any=FAKE, out=FAKE, out_lo=FAKE,
            stats=FAKE, **{f"{n}_stride{i}": 64 for n in ("q", "k", "v", "out") for i in range(3)},
            scale=0.1, index_batch=2, batch=2, heads=4, kv_heads=2, queries=100, keys=100, head_dim=64, buckets=6,
            dtype=_native.MF_DTYPE_BF16, table_dtype=0)
ATTN_REFUSALS = [(dict(q=None), INVALID, "non-NULL"), (dict(query_any=None), INVALID, "non-NULL"),
                 (dict(queries=-1), INVALID, "non-negative"), (dict(dtype=0), UNSUPPORTED, "float16/bfloat16"),
                 (dict(table_dtype=7), UNSUPPORTED, "table"), (dict(head_dim=36), UNSUPPORTED, "head_dim"),
                 (dict(head_dim=136), UNSUPPORTED, "head_dim"), (dict(buckets=65), UNSUPPORTED, "[1, 64]"),
                 (dict(scale=math.nan), INVALID, "finite"), (dict(index_batch=3), INVALID, "index_batch"),
                 (dict(keys=2 ** 24 + 1), UNSUPPORTED, "2^24"), (dict(kv_heads=3), UNSUPPORTED, "divide"),
                 (dict(kv_heads=0), UNSUPPORTED, "divide"), (dict(heads=66, kv_heads=2), UNSUPPORTED, "at most 32"),
                 (dict(k=FAKE + 8), INVALID, "aligned"), (dict(v_stride1=4), INVALID, "multiples of 8"),
                 (dict(q_stride2=-8), INVALID, "multiples of 8"), (dict(k_stride2=2 ** 23), UNSUPPORTED, "2^23")]


def test_attention_entries_refuse_before_any_device_call():
    lib = _native.lib()
    forward = lambda **kw: _native.MfBucketAttnArgs(**(ATTN | kw))

    def backward(bwd=None, **kw):
        a = dict(fwd=forward(**kw), index_t=FAKE, grad_out=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, dtable=FAKE,
                 **{f"{n}_stride{i}": 64 for n in ("grad_out", "dq", "dk", "dv") for i in range(3)})
        a.update(bwd or {})
        return _native.MfBucketAttnBwdArgs(**a)

    for fn, make in ((lib.mf_bucket_attn, forward), (lib.mf_bucket_attn_bwd, backward)):
        refused(fn, None, INVALID, "args is NULL")
        for kw, status, match in ATTN_REFUSALS:
            refused(fn, make(**kw), status, match)
        assert fn(make(batch=0, index_batch=1), None) == _native.MF_OK
    few = dict(queries=1, keys=5000)
    need = lib.mf_bucket_attn_workspace_size(forward(**few))
    assert need > 0 and lib.mf_bucket_attn_workspace_size(forward(queries=2000, batch=64, index_batch=1)) == 0
    refused(lib.mf_bucket_attn, forward(**few), INVALID, "workspace")
    refused(lib.mf_bucket_attn, forward(**few, workspace=FAKE, workspace_bytes=need - 1), INVALID, "workspace")
    refused(lib.mf_bucket_attn, forward(batch=2 ** 24, index_batch=1, heads=32, kv_heads=32), UNSUPPORTED, "too large")
    for bwd, status, match in ((dict(index_t=None), INVALID, "non-NULL"), (dict(dv=None), INVALID, "non-NULL"),
                               (dict(dq=FAKE + 8), INVALID, "aligned"), (dict(dk_stride2=7), INVALID, "multiples of 8"),
                               (dict(grad_out_stride2=2 ** 23), UNSUPPORTED, "2^23"), (dict(), INVALID, "workspace")):
        refused(lib.mf_bucket_attn_bwd, backward(bwd), status, match)
    refused(lib.mf_bucket_attn_bwd, backward(stats=None), INVALID, "non-NULL")
    refused(lib.mf_bucket_attn_bwd, backward(keys=0), UNSUPPORTED, "positive")
    refused(lib.mf_bucket_attn_bwd, backward(batch=2 ** 23, index_batch=1), UNSUPPORTED, "too large")
    plain, sums = (lib.mf_bucket_attn_bwd_workspace_size(backward(b)) for b in (dict(dtable=None), None))
    half = lib.mf_bucket_attn_bwd_workspace_size(backward(dtype=_native.MF_DTYPE_F16))
    assert 0 < plain < sums < half
    assert lib.mf_bucket_attn_bwd_workspace_size(backward(queries=0)) == 0


def test_counts_past_32_bits_are_refused():
    """(zero-stride views: nothing of that size is allocated)"""
    from matterformer_amd import pair_buckets

    for counts in ((2 ** 32 + 5, 1, 1), (1, 2 ** 31, 1), (1, 1, 2 ** 32 + 1)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            pair_buckets._launch(0, *counts, torch.device("cpu"), buckets=1, gradients=False, symmetric=False)


def test_offset_edges_of_the_c_entry_are_whole():
    """(between whole numbers, an edge's side would hang on the path that a tile takes)"""
    lib = _native.lib()

    def args(*edges, **kw):
        held.append((ctypes.c_double * len(edges))(*edges))
        return _native.MfPairBucketsArgs(query_pos=FAKE, key_pos=2 * FAKE, edges=ctypes.addressof(held[-1]), index=FAKE,
                                         index_t=2 * FAKE, key_any=3 * FAKE, query_any=4 * FAKE, cutoff=-1.0,
                                         source=_native.MF_BUCKETS_OFFSET, num_edges=len(edges), buckets=len(edges) + 1,
                                         batch=kw.get("batch", 1), queries=5, keys=5)

    held = []
    for edges in ((0.5,), (0.2, 0.7), (-3.0, 2.0 ** 51 + 0.5), (-0.25, 0.0)):
        refused(lib.mf_pair_buckets, args(*edges), INVALID, "whole")
    assert lib.mf_pair_buckets(args(-(2.0 ** 53), -1.0, 0.0, 2.0 ** 53, batch=0), None) == _native.MF_OK


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_torch_formulation_is_fp32_under_autocast(dtype):
    """Autocast would take its products in 16 bits, forward and backward."""
    torch.manual_seed(12)
    buckets = index_buckets(torch.randint(-1, 4, (2, 9, 11)), 4)
    q, k, v = (torch.randn(2, 4, n, 8).to(dtype) for n in (9, 11, 11))
    table, go = torch.randn(4, 4), torch.randn(2, 4, 9, 8).to(dtype)
    results = []
    for on in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, table)]
        with torch.autocast("cpu", dtype=torch.bfloat16, enabled=on):
            out, lse = bucket_attention_torch(*leaves, buckets, 0.35)
        assert out.dtype == dtype and lse.dtype == torch.float32
        results.append([out, lse, *torch.autograd.grad((out, lse), leaves, (go, torch.ones_like(lse)))])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_empty_calls_are_zeros_with_gradients():
    for B, H, Nq, Nk in ((0, 2, 5, 5), (2, 0, 5, 5), (2, 2, 0, 5), (2, 2, 5, 0)):
        q, k, v = (torch.randn(B, H, n, 8, requires_grad=True) for n in (Nq, Nk, Nk))
        table = torch.randn(4, H, requires_grad=True)
        out, lse = bucket_attention(q, k, v, table, index_buckets(torch.zeros(B, Nq, Nk, dtype=torch.int32), 4),
                                    return_lse=True)
        assert out.shape == q.shape and not out.any() and lse.shape == q.shape[:3] and not lse.any()
        for t, up in ((out, torch.ones_like(out)), (lse, torch.ones_like(lse))):
            grads = torch.autograd.grad(t, (q, k, v, table), up, retain_graph=True, allow_unused=True)
            assert all(g is None or g.shape == x.shape and not g.any() for g, x in zip(grads, (q, k, v, table)))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64,
                                   torch.uint64])
def test_indexes_of_every_whole_type(dtype):
    """Numbers past 32 bits leave the pair out, whatever their low bits."""
    top = torch.iinfo(dtype).max
    numbers = [n for n in (0, 3, 4, 63, 64, 127, 255, 256, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 63 - 1, 2 ** 63, 2 ** 64 - 1, top)
               if n <= top]
    index = torch.tensor(numbers, dtype=dtype).view(1, 1, -1)
    want = [n if n < 4 else MASKED for n in numbers]
    assert index_buckets(index, 4).index.flatten().tolist() == want
    if dtype.is_signed:
        assert index_buckets(torch.tensor([[[-1, torch.iinfo(dtype).min]]], dtype=dtype), 4).index.eq(MASKED).all()


def test_a_negative_batch_of_the_bias_is_refused():
    b = index_buckets(torch.zeros(1, 3, 5, dtype=torch.int32), 4)
    for n in (-1, -3):
        with pytest.raises(ValueError, match="batch"):
            bucket_bias(torch.zeros(4, 2), b, batch=n)
    assert bucket_bias(torch.zeros(4, 2), b, batch=0).shape == (0, 2, 3, 5)


@pytest.mark.parametrize("causal", [False, True])
def test_offset_edges_end_at_the_greatest_offset(causal):
    """Offsets from max_offset on share the last bucket, and none before does (of sides with widening buckets)."""
    for n in (4, 5, 14, 27, 33, 64):
        for most in (63, 115, 122, 230, 237, 512, 1000, 4096, 99999, 2 ** 31, 2 ** 53):
            edges = offset_edges(n, most, causal=causal)
            assert all(a < b for a, b in zip(edges, edges[1:])) and 1 - edges[0] == most, (n, most)
            assert causal or n < 5 or edges[-1] == most, (n, most)
