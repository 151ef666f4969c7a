"""Buckets of the pairs of a batch and the learned bias they give.

  PairBuckets       which of at most 64 buckets every pair (query, key) has, or that it is left out; made once for a
                    batch and shared by its heads and layers, in the layout the kernels read
  distance_buckets  by the distance of two atoms (NonPeriodicGeometryAdapter.forward's pair distance,
                    src/matterformer/geometry/adapters.py:98-100)
  offset_buckets    by the offset of a key's place in a sequence from its query's
  value_buckets     by any number of the pair: a geometry adapter's pair_dist, periodic ones too
  index_buckets     given as they are
  offset_edges      edges of offset buckets: one by one near zero, then wider by a constant factor
  bucket_bias       table[bucket(i, j), h] for every pair and head: an attn_head_bias
                    (src/matterformer/models/transformer.py:256-268) or a term of a SimplicialFactorizedBias
                    (src/matterformer/models/simplicial_attention.py:18-47), with the table's gradient

Edges e_0 < e_1 < .. rise, and a pair's bucket is how many of them are at or below its value, so there is one bucket
more than edges.  GPU tensors run mf_pair_buckets, mf_bucket_bias and mf_bucket_bias_bwd (csrc/pair_buckets.hip); a
missing library raises.  CPU tensors, and calls with use_hip=False, take the torch formulation.
"""

from __future__ import annotations

import math
import operator
from array import array
from typing import Iterable

import torch
from torch.autograd.function import once_differentiable

from matterformer_amd import _native

MAX_BUCKETS = _native.MF_MAX_BUCKETS
MASKED = _native.MF_BUCKET_MASKED  # the index of a pair that is left out
TILE = 64

_TABLE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


class PairBuckets:
    """The buckets of a batch's pairs.  ``index`` (B, Nq, Nk) uint8: 0 .. num_buckets - 1, or MASKED; ``index_t`` its
    transpose, kept for gradients (None without).  A batch of one serves any batch.  On the GPU both are views of rows
    padded to 64 bytes, and key_any, query_any say which keys and queries of each 64 x 64 tile have a pair.  The tensors
    are not to be changed."""

    def __init__(self, index: torch.Tensor, index_t: torch.Tensor | None, num_buckets: int,
                 key_any: torch.Tensor | None = None, query_any: torch.Tensor | None = None) -> None:
        self.index = index
        self.index_t = index_t
        self.num_buckets = int(num_buckets)
        self.key_any = key_any
        self.query_any = query_any
        self._laid_out = False  # as the kernels read it (check_layout)

    @property
    def batch(self) -> int:
        return self.index.shape[0]

    @property
    def queries(self) -> int:
        return self.index.shape[1]

    @property
    def keys(self) -> int:
        return self.index.shape[2]

    @property
    def device(self) -> torch.device:
        return self.index.device

    def allowed(self) -> torch.Tensor:
        """(B, Nq, Nk) bool: the pairs that count."""
        return self.index != MASKED


def _round_edges(edges, whole: bool) -> array:
    """The edges as host numbers: whole ones, or rounded to fp32 as the values they are compared with."""
    if isinstance(edges, torch.Tensor):
        if edges.device.type != "cpu" or edges.ndim != 1:
            raise ValueError("edges must be a sequence of numbers or a 1-D CPU tensor")
        edges = edges.tolist()
    if len(edges) > MAX_BUCKETS - 1:
        raise ValueError(f"at most {MAX_BUCKETS - 1} edges, got {len(edges)}")
    if whole:
        try:
            edges = array("q", edges)
        except OverflowError:
            raise ValueError("edges of offsets must not pass 2^53") from None
        except TypeError:  # not integers: whole floats pass
            if any(not math.isfinite(e) or e != math.floor(e) for e in edges):
                raise ValueError("edges of offsets must be finite and whole numbers") from None
    else:
        edges = array("f", edges)  # (past fp32's range becomes infinite)
    out = array("d", edges)
    if out and not (all(map(operator.lt, out, out[1:])) and math.isfinite(out[0]) and math.isfinite(out[-1])):
        raise ValueError("edges must be finite and rise")
    if whole and out and max(-edges[0], edges[-1]) > 2 ** 53:
        raise ValueError("edges of offsets must not pass 2^53")
    return out


def _distance_edges(edges) -> array:
    out = _round_edges(edges, whole=False)
    if out and out[0] < 0.0:
        raise ValueError("edges of distances must not be negative")
    return out


def check_edges(edges, *, distances: bool, cutoff: float | None = None) -> list[float]:
    """The edges of distance_buckets, or of value_buckets, as a list; what those refuse is refused."""
    edges = [float(e) for e in edges]
    _distance_edges(edges) if distances else _round_edges(edges, whole=False)
    _check_cutoff(cutoff)
    return edges


def _pad_bytes(pad: torch.Tensor | None, B: int, N: int, name: str, device: torch.device) -> torch.Tensor | None:
    if pad is None:
        return None
    if pad.shape != (B, N):
        raise ValueError(f"{name} must have shape ({B}, {N}), got {tuple(pad.shape)}")
    if pad.device != device:
        raise RuntimeError("all tensors must be on the same device")
    pad = pad.contiguous()
    return pad.view(torch.uint8) if pad.dtype == torch.bool else pad.ne(0).view(torch.uint8)


def _check_counts(*counts: int) -> None:
    if any(n >= 1 << 31 for n in counts):  # before they are cut to 32 bits
        raise RuntimeError(f"pair buckets support counts below 2^31, got {counts}")


def _launch(source: int, B: int, Nq: int, Nk: int, device: torch.device, *, edges=None, buckets: int,
            query_pos=None, key_pos=None, query_step: int = 0, key_step: int = 0, values=None, query_pad=None,
            key_pad=None, cutoff: float = -1.0, causal: bool = False, gradients: bool, symmetric: bool) -> PairBuckets:
    _check_counts(B, Nq, Nk)
    S, St = (Nk + 63) // 64 * 64, (Nq + 63) // 64 * 64
    TQ, TK = St // TILE, S // TILE
    index = torch.empty(B, Nq, S, dtype=torch.uint8, device=device)
    key_any = torch.empty(B, TQ, TK, dtype=torch.int64, device=device)
    if symmetric:
        index_t, query_any = index, key_any
    elif gradients:
        index_t = torch.empty(B, Nk, St, dtype=torch.uint8, device=device)
        query_any = torch.empty(B, TK, TQ, dtype=torch.int64, device=device)
    else:
        index_t, query_any = None, torch.empty(B, TK, TQ, dtype=torch.int64, device=device)
    if B * Nq * Nk > 0:
        args = _native.MfPairBucketsArgs(
            query_pos=_native.ptr(query_pos), key_pos=_native.ptr(key_pos), values=_native.ptr(values),
            query_pad=_native.ptr(query_pad), key_pad=_native.ptr(key_pad),
            edges=edges.buffer_info()[0] if edges else None, index=index.data_ptr(),
            index_t=_native.ptr(index_t), key_any=key_any.data_ptr(), query_any=query_any.data_ptr(),
            query_step=query_step, key_step=key_step, cutoff=cutoff, source=source,
            num_edges=0 if edges is None else len(edges), buckets=buckets, causal=int(causal), batch=B, queries=Nq,
            keys=Nk)
        _native.launch("mf_pair_buckets", args, device)
    view_t = None if index_t is None else index_t[:, :, :Nq]
    made = PairBuckets(index[:, :, :Nk], view_t, buckets, key_any, query_any)
    made._laid_out = True
    return made


def _from_torch(index: torch.Tensor, buckets: int, allowed: torch.Tensor | None, query_pad, key_pad,
                gradients: bool) -> PairBuckets:
    """The torch formulation's end: masks applied."""
    index = index.to(torch.uint8)
    drop = torch.zeros_like(index, dtype=torch.bool) if allowed is None else ~allowed
    if key_pad is not None:
        drop = drop | key_pad[:, None, :].bool()
    if query_pad is not None:
        drop = drop | query_pad[:, :, None].bool()
    index = index.masked_fill(drop, MASKED)
    return PairBuckets(index, index.transpose(1, 2).contiguous() if gradients else None, buckets)


def _count_edges(values: torch.Tensor, edges: Iterable[float]) -> torch.Tensor:
    index = torch.zeros(values.shape, dtype=torch.uint8, device=values.device)
    for e in edges:
        index += values >= e
    return index


def _check_cutoff(cutoff: float | None) -> float:
    """The cutoff in fp32, or -1 for none."""
    if cutoff is None:
        return -1.0
    cutoff = float(cutoff)
    if not 0.0 <= cutoff < math.inf:
        raise ValueError(f"cutoff must be finite and not negative, got {cutoff}")
    return array("f", [min(cutoff, 3.4028234663852886e38)])[0]


def distance_buckets(coords: torch.Tensor, edges, *, pad_mask: torch.Tensor | None = None,
                     cutoff: float | None = None, use_hip: bool = True) -> PairBuckets:
    """Buckets of the distances of every two atoms: how many of the rising ``edges`` (fp32, not negative) are at or below
    |x_i - x_j|.  coords (B, N, 3), taken in fp32; pad_mask (B, N), True = padding, whose pairs are left out, as are those
    further apart than ``cutoff``.  Squares are compared, in fp64: a distance at an edge falls on its exact side.  (An atom
    whose coordinates are NaN has bucket 0 with every other.)  The matrix is its own transpose.  ``use_hip`` = False takes
    the torch formulation for GPU tensors too; its buckets are for bucket_attention_torch, the kernels refuse them."""
    if coords.ndim != 3 or coords.shape[-1] != 3:
        raise ValueError(f"coords must have shape (B, N, 3), got {tuple(coords.shape)}")
    host = _distance_edges(edges)
    cut = _check_cutoff(cutoff)
    B, N, _ = coords.shape
    dev = coords.device
    pad = _pad_bytes(pad_mask, B, N, "pad_mask", dev)
    c = coords.detach().float().contiguous()
    if dev.type == "cuda" and use_hip:
        return _launch(_native.MF_BUCKETS_DISTANCE, B, N, N, dev, edges=host, buckets=len(host) + 1, query_pos=c,
                       key_pos=c, query_step=3 * N, key_step=3 * N, query_pad=pad, key_pad=pad, cutoff=cut,
                       gradients=True, symmetric=True)
    d = c.double()[:, :, None] - c.double()[:, None]
    d2 = (d[..., 0] * d[..., 0] + d[..., 1] * d[..., 1]) + d[..., 2] * d[..., 2]
    index = _count_edges(d2, [e * e for e in host])
    return _from_torch(index, len(host) + 1, None if cutoff is None else ~(d2 > cut * cut), pad, pad, True)


def offset_buckets(query_positions: torch.Tensor, key_positions: torch.Tensor, edges, *,
                   pad_mask: torch.Tensor | None = None, query_pad_mask: torch.Tensor | None = None,
                   causal: bool = False, gradients: bool = True) -> PairBuckets:
    """Buckets of the offsets key position - query position: how many of the rising whole ``edges`` are at or below it.
    Positions are whole, (B, N) or (N,) for every batch entry, and need not follow one another.  pad_mask (B, Nk) and
    query_pad_mask (B, Nq), True = padding: their pairs are left out; ``causal``: so are keys at a later position than
    the query's.  Positions are 64-bit and their differences must be too.  ``gradients`` = False leaves out what only
    gradients read (a new token's step).  Positions and pads without a batch give buckets of a batch of one, which serve
    any batch."""
    host = _round_edges(edges, whole=True)
    positions = []
    for name, p in (("query_positions", query_positions), ("key_positions", key_positions)):
        if p.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
            raise RuntimeError(f"{name} must be whole numbers, got {p.dtype}")
        if p.ndim not in (1, 2):
            raise ValueError(f"{name} must have shape (B, N) or (N,), got {tuple(p.shape)}")
        p = p if p.ndim == 2 else p[None]
        p = p.to(torch.int64)
        positions.append(p if p.stride(1) == 1 or p.shape[1] <= 1 else p.contiguous())
    qp, kp = positions
    dev = qp.device
    if kp.device != dev:
        raise RuntimeError("all tensors must be on the same device")
    B = max(t.shape[0] for t in (qp, kp, pad_mask, query_pad_mask) if t is not None)
    if any(t.shape[0] == 0 for t in (qp, kp)):
        B = 0
    for name, p in (("query_positions", qp), ("key_positions", kp)):
        if p.shape[0] not in (1, B):
            raise ValueError(f"{name} must have {B} rows or one, got {p.shape[0]}")
    Nq, Nk = qp.shape[1], kp.shape[1]
    kpad = _pad_bytes(pad_mask, B, Nk, "pad_mask", dev)
    qpad = _pad_bytes(query_pad_mask, B, Nq, "query_pad_mask", dev)
    if dev.type == "cuda":
        return _launch(_native.MF_BUCKETS_OFFSET, B, Nq, Nk, dev, edges=host, buckets=len(host) + 1, query_pos=qp,
                       key_pos=kp, query_step=qp.stride(0) if qp.shape[0] > 1 else 0,
                       key_step=kp.stride(0) if kp.shape[0] > 1 else 0, query_pad=qpad, key_pad=kpad, causal=causal,
                       gradients=gradients, symmetric=False)
    offset = (kp[:, None, :] - qp[:, :, None]).expand(B, Nq, Nk)
    # (compared as whole numbers: a float would round the far ones)
    return _from_torch(_count_edges(offset, map(int, host)), len(host) + 1, offset <= 0 if causal else None, qpad, kpad,
                       gradients)


def value_buckets(values: torch.Tensor, edges, *, pad_mask: torch.Tensor | None = None,
                  query_pad_mask: torch.Tensor | None = None, cutoff: float | None = None,
                  gradients: bool = True, use_hip: bool = True) -> PairBuckets:
    """Buckets of given numbers (B, Nq, Nk), taken in fp32: how many of the rising ``edges`` (fp32) are at or below each.
    Pairs of padding (pad_mask (B, Nk), query_pad_mask (B, Nq)) and those above ``cutoff`` are left out; NaN has bucket 0.
    ``use_hip`` as in distance_buckets."""
    if values.ndim != 3:
        raise ValueError(f"values must have shape (B, Nq, Nk), got {tuple(values.shape)}")
    host = _round_edges(edges, whole=False)
    cut = _check_cutoff(cutoff)
    B, Nq, Nk = values.shape
    dev = values.device
    kpad = _pad_bytes(pad_mask, B, Nk, "pad_mask", dev)
    qpad = _pad_bytes(query_pad_mask, B, Nq, "query_pad_mask", dev)
    v = values.detach().float().contiguous()
    if dev.type == "cuda" and use_hip:
        return _launch(_native.MF_BUCKETS_VALUE, B, Nq, Nk, dev, edges=host, buckets=len(host) + 1, values=v,
                       query_pad=qpad, key_pad=kpad, cutoff=cut, gradients=gradients, symmetric=False)
    return _from_torch(_count_edges(v, host), len(host) + 1, None if cutoff is None else ~(v > cut), qpad, kpad, gradients)


def index_buckets(index: torch.Tensor, num_buckets: int, *, pad_mask: torch.Tensor | None = None,
                  query_pad_mask: torch.Tensor | None = None, gradients: bool = True) -> PairBuckets:
    """Buckets given as they are: whole numbers (B, Nq, Nk); those below 0 or from num_buckets on leave the pair out."""
    if index.ndim != 3 or index.is_floating_point() or index.is_complex() or index.dtype == torch.bool:
        raise ValueError(f"index must be whole numbers of shape (B, Nq, Nk), got {index.dtype} {tuple(index.shape)}")
    if not 1 <= int(num_buckets) <= MAX_BUCKETS:
        raise ValueError(f"num_buckets must be in [1, {MAX_BUCKETS}], got {num_buckets}")
    B, Nq, Nk = index.shape
    dev = index.device
    kpad = _pad_bytes(pad_mask, B, Nk, "pad_mask", dev)
    qpad = _pad_bytes(query_pad_mask, B, Nq, "query_pad_mask", dev)
    if index.dtype in (torch.int64, torch.uint64):
        index = index.to(torch.int64).clamp(-1, MAX_BUCKETS)  # before it is cut to 32 bits (from 2^63 on: negative)
    i = index.to(torch.int32).contiguous()
    if dev.type == "cuda":
        return _launch(_native.MF_BUCKETS_INDEX, B, Nq, Nk, dev, buckets=int(num_buckets), values=i, query_pad=qpad,
                       key_pad=kpad, gradients=gradients, symmetric=False)
    allowed = (i >= 0) & (i < int(num_buckets))
    return _from_torch(i.clamp(0, MAX_BUCKETS), int(num_buckets), allowed, qpad, kpad, gradients)


def offset_edges(num_buckets: int, max_offset: int, *, causal: bool = False) -> list[int]:
    """Rising edges of ``num_buckets`` offset buckets: one bucket an offset near zero (half of a side's), then buckets that
    widen by a constant factor up to ``max_offset``, beyond which all share the last.  Keys before and after the query
    have buckets of their own unless ``causal``, where only those before it do."""
    num_buckets, max_offset = int(num_buckets), int(max_offset)
    if not 1 <= num_buckets <= MAX_BUCKETS:
        raise ValueError(f"num_buckets must be in [1, {MAX_BUCKETS}], got {num_buckets}")
    before = num_buckets - 1 if causal else num_buckets // 2
    after = 0 if causal else num_buckets - 1 - before
    if max_offset < max(before, after):
        raise ValueError(f"max_offset must be at least {max(before, after)}, got {max_offset}")

    def steps(n: int) -> list[int]:
        near = (n + 1) // 2
        out = list(range(1, near + 1))
        while len(out) < n:
            if len(out) + 1 == n:
                at = max_offset
            else:
                at = near * (max_offset / near) ** ((len(out) + 1 - near) / (n - near))
            out.append(max(out[-1] + 1, min(int(at), max_offset - (n - 1 - len(out)))))
        return out

    # offsets of -s and less lie below the edge 1 - s
    return [1 - s for s in reversed(steps(before))] + steps(after)


def _check_table(table: torch.Tensor, buckets: PairBuckets) -> None:
    if not isinstance(buckets, PairBuckets):
        raise TypeError(f"buckets must be PairBuckets, got {type(buckets).__name__}")
    if table.ndim != 2 or table.shape[0] != buckets.num_buckets:
        raise ValueError(f"table must have shape ({buckets.num_buckets}, heads), got {tuple(table.shape)}")
    if table.device != buckets.device:
        raise RuntimeError("all tensors must be on the same device")


def check_layout(buckets: PairBuckets) -> None:
    """The kernels read the buckets by address: their types and layout."""
    if buckets._laid_out:
        return
    B, Nq, Nk = buckets.index.shape
    S, St = (Nk + 63) // 64 * 64, (Nq + 63) // 64 * 64
    TQ, TK = St // TILE, S // TILE
    ok = buckets.key_any is not None and buckets.query_any is not None
    for t, shape, pitch in ((buckets.index, (B, Nq, Nk), S), (buckets.index_t, (B, Nk, Nq), St)):
        if t is not None and t.numel() > 0:
            ok = ok and t.dtype == torch.uint8 and t.shape == shape and t.device == buckets.device \
                and t.stride() == (shape[1] * pitch, pitch, 1) and t.data_ptr() % 16 == 0
    for t, shape in ((buckets.key_any, (B, TQ, TK)), (buckets.query_any, (B, TK, TQ))):
        ok = ok and t.dtype == torch.int64 and t.shape == shape and t.device == buckets.device and t.is_contiguous()
    if not ok:
        raise ValueError("buckets must be as distance_buckets, offset_buckets, value_buckets or index_buckets make them")
    buckets._laid_out = True


def table_with_masked(table: torch.Tensor) -> torch.Tensor:
    """The table with a row of -inf for the pairs that are left out, which ``table_rows`` gives."""
    return torch.cat([table, table.new_full((1, table.shape[1]), -math.inf)])


def table_rows(buckets: PairBuckets) -> torch.Tensor:
    """(B, Nq, Nk) int64 rows of table_with_masked."""
    return torch.where(buckets.index == MASKED, buckets.num_buckets, buckets.index.long())


def _bias_args(buckets: PairBuckets, batch: int, heads: int, table_dtype: torch.dtype, bias: torch.Tensor, **kw):
    return _native.MfBucketBiasArgs(
        index=buckets.index.data_ptr(), bias=bias.data_ptr(), index_batch=buckets.batch, batch=batch, heads=heads,
        queries=buckets.queries, keys=buckets.keys, buckets=buckets.num_buckets,
        table_dtype=_native.dtype_code(table_dtype), bias_dtype=_native.dtype_code(bias.dtype), **kw)


def _bias_forward(table: torch.Tensor, buckets: PairBuckets, batch: int, dtype: torch.dtype) -> torch.Tensor:
    H = table.shape[1]
    bias = torch.empty(batch, H, buckets.queries, buckets.keys, dtype=dtype, device=table.device)
    if bias.numel() > 0:
        t = table.contiguous()
        _native.launch("mf_bucket_bias", _bias_args(buckets, batch, H, t.dtype, bias, table=t.data_ptr()), table.device)
    return bias


class _BucketBiasFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets, batch, dtype):
        ctx.buckets, ctx.batch, ctx.heads, ctx.table_dtype = buckets, batch, table.shape[1], table.dtype
        return _bias_forward(table, buckets, batch, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        buckets = ctx.buckets
        dtable = torch.empty(buckets.num_buckets, ctx.heads, dtype=ctx.table_dtype, device=grad.device)
        if grad.numel() == 0:
            return dtable.zero_(), None, None, None
        g = grad.contiguous()
        if g.data_ptr() % 16:
            g = g.clone()
        args = _bias_args(buckets, ctx.batch, ctx.heads, ctx.table_dtype, g, dtable=dtable.data_ptr())
        nbytes = int(_native.lib().mf_bucket_bias_bwd_workspace_size(args))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=grad.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
        _native.launch("mf_bucket_bias_bwd", args, grad.device)
        return dtable, None, None, None


def bucket_bias(table: torch.Tensor, buckets: PairBuckets, *, batch: int | None = None,
                dtype: torch.dtype | None = None) -> torch.Tensor:
    """bias (B, H, Nq, Nk) = table[bucket(i, j), h], -inf where the pair is left out.

    table (num_buckets, H), fp32, fp16 or bf16, H <= 128; ``dtype`` of the bias (the table's unless given).  ``batch``
    repeats the buckets of a batch of one.  Differentiable in the table: the sums of the bias's gradient by bucket, in
    fp32 in a fixed order.  Entries of the bias at pairs that are left out take no gradient."""
    _check_table(table, buckets)
    B = buckets.batch if batch is None else int(batch)
    if B < 0 or (B != buckets.batch and buckets.batch != 1):
        raise ValueError(f"batch must be {buckets.batch if buckets.batch != 1 else 'not negative'}, got {B}")
    dtype = table.dtype if dtype is None else dtype
    if table.device.type != "cuda":
        bias = table_with_masked(table)[table_rows(buckets)].permute(0, 3, 1, 2).to(dtype)
        return bias.expand(B, *bias.shape[1:]).contiguous()
    if table.dtype not in _TABLE_DTYPES or dtype not in _TABLE_DTYPES:
        raise RuntimeError(f"bucket_bias only supports float32/float16/bfloat16, got {table.dtype} and {dtype}")
    if table.shape[1] > 128:
        raise RuntimeError(f"bucket_bias supports up to 128 heads, got {table.shape[1]}")
    _check_counts(B, buckets.queries, buckets.keys)
    check_layout(buckets)
    if _native.takes_gradient(table):
        return _BucketBiasFunction.apply(table, buckets, B, dtype)
    return _bias_forward(table, buckets, B, dtype)
