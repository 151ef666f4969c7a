"""Attention over all pairs with a learned bias by buckets:

  out_i = sum_j softmax_j(scale q_i . k_j + table[bucket(i, j), h]) v_j    over the pairs that are not left out

the reference's pairwise attention with an attn_head_bias (src/matterformer/models/transformer.py:256-268,
src/matterformer/models/regular_attention.py:262-268,303-308), where the bias is a table of learned numbers by bucket
(pair_buckets).  The bias is never written out: the kernels read a byte a pair, shared by the heads and layers.

GPU tensors run mf_bucket_attn and, for the gradients of q, k, v and the table, mf_bucket_attn_bwd, which forms the
probabilities again (csrc/bucket_attn.hip, bucket_attn_bwd.hip); a missing library raises.  CPU tensors take the torch
formulation.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from matterformer_amd import _native
from matterformer_amd.pair_buckets import PairBuckets, _check_table, check_layout, table_rows, table_with_masked

_TABLE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    """Elements from one batch entry, head and token to the next (0 where there is only one)."""
    n, s = t.shape, t.stride()
    return (s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


def _rows_apart(t: torch.Tensor) -> bool:
    """A head's entries next to one another, the rest by steps that the kernels take."""
    b, h, n = _strides(t)
    return t.stride(3) == 1 and b % 8 == 0 and h % 8 == 0 and n % 8 == 0 and min(b, h, n) >= 0 and n < 1 << 23


def _readable(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0 and _rows_apart(t)


def _operand(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it: itself, or a copy."""
    if _readable(t):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _like(t: torch.Tensor) -> torch.Tensor:
    """An output in t's layout (heads of projected rows come back as such views)."""
    out = torch.empty_like(t)
    return out if _rows_apart(out) else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _arguments(q, k, v, table, buckets: PairBuckets, out, out_lo, lse, stats, scale: float):
    B, H, Nq, D = q.shape
    ptr = _native.ptr
    return _native.MfBucketAttnArgs(  # in the order of the fields, which is quicker than by name
        q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), buckets.index.data_ptr(),
        buckets.key_any.data_ptr(), buckets.query_any.data_ptr(), out.data_ptr(), ptr(out_lo), ptr(lse), ptr(stats), None,
        0, *_strides(q), *_strides(k), *_strides(v), *_strides(out), scale, buckets.index.shape[0], B, H, k.shape[1], Nq,
        k.shape[2], D, buckets.num_buckets, _native.dtype_code(q.dtype), _native.dtype_code(table.dtype))


def _forward(q, k, v, table, buckets, scale: float, *, lse: bool, training: bool):
    """out, lse, and for gradients what out's rounding left, the rows' maxima and sums and the call's arguments (None where
    not asked)."""
    B, H, Nq, D = q.shape
    out = _like(q)
    lse_out = torch.empty(B, H, Nq, dtype=torch.float32, device=q.device) if lse else None
    lo = torch.empty(B, H, Nq, D, dtype=q.dtype, device=q.device) if training else None
    stats = torch.empty(2, B, H, Nq, dtype=torch.float32, device=q.device) if training else None
    if q.numel() == 0 or k.numel() == 0:
        for t in (out, lse_out, lo, stats):
            if t is not None:
                t.zero_()
        return out, lse_out, lo, stats, None
    args = _arguments(q, k, v, table, buckets, out, lo, lse_out, stats, scale)
    nbytes = int(_native.lib().mf_bucket_attn_workspace_size(args))
    if nbytes > 0:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
    _native.launch("mf_bucket_attn", args, q.device)
    return out, lse_out, lo, stats, args


class _BucketAttentionFunction(torch.autograd.Function):
    """mf_bucket_attn with mf_bucket_attn_bwd: differentiable in q, k, v and the table through out and lse."""

    @staticmethod
    def forward(ctx, q, k, v, table, buckets, scale):
        out, lse, lo, stats, args = _forward(q, k, v, table, buckets, scale, lse=True, training=True)
        ctx.save_for_backward(q, k, v, table, out, lo, stats)
        ctx.buckets, ctx.args = buckets, args
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_lse):
        if grad_out is None and grad_lse is None:
            return (None,) * 6
        q, k, v, table, out, lo, stats = ctx.saved_tensors
        q, k, v, out = _operand(q), _operand(k), _operand(v), _operand(out)
        buckets = ctx.buckets
        go = torch.zeros_like(out) if grad_out is None else _operand(grad_out)
        gl = None if grad_lse is None else grad_lse.contiguous()
        dq, dk, dv = (_like(t) for t in (q, k, v))
        dtable = torch.empty_like(table) if ctx.needs_input_grad[3] else None
        if q.numel() == 0 or k.numel() == 0:
            for t in (dq, dk, dv, dtable):
                if t is not None:
                    t.zero_()
            return dq, dk, dv, dtable, None, None
        args = _native.MfBucketAttnBwdArgs(
            ctx.args, buckets.index_t.data_ptr(), go.data_ptr(), _native.ptr(gl), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), _native.ptr(dtable), None, 0, *_strides(go), *_strides(dq), *_strides(dk), *_strides(dv))
        f = args.fwd  # a copy; the saved tensors may have been moved meanwhile (saved tensor hooks), and laid out anew
        f.q, f.k, f.v, f.table = q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr()
        f.out, f.out_lo, f.stats = out.data_ptr(), lo.data_ptr(), stats.data_ptr()
        f.q_stride0, f.q_stride1, f.q_stride2 = _strides(q)
        f.k_stride0, f.k_stride1, f.k_stride2 = _strides(k)
        f.v_stride0, f.v_stride1, f.v_stride2 = _strides(v)
        f.out_stride0, f.out_stride1, f.out_stride2 = _strides(out)
        nbytes = int(_native.lib().mf_bucket_attn_bwd_workspace_size(args))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
        _native.launch("mf_bucket_attn_bwd", args, q.device)
        return dq, dk, dv, dtable, None, None


def _check_operands(q, k, v, table, buckets: PairBuckets) -> None:
    if q.ndim != 4 or k.ndim != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError("q must have shape (B, H, Nq, D), k and v (B, KV, Nk, D)")
    _check_table(table, buckets)
    B, H, Nq, D = q.shape
    KV, Nk = k.shape[1:3]
    if table.shape[1] != H:
        raise ValueError(f"table must have shape ({buckets.num_buckets}, {H}), got {tuple(table.shape)}")
    if buckets.batch not in (1, B) or (buckets.queries, buckets.keys) != (Nq, Nk):
        raise ValueError(f"buckets must be of ({B}, {Nq}, {Nk}) pairs, got {tuple(buckets.index.shape)}")
    if (KV == 0) != (H == 0) or (KV and H % KV):
        raise ValueError(f"the heads of k and v must divide those of q, got {KV} and {H}")
    if any(t.device != q.device for t in (k, v, table)):
        raise RuntimeError("all tensors must be on the same device")


def bucket_attention_torch(q, k, v, table, buckets: PairBuckets, scale: float, *, dropout: float = 0.0):
    """out and lse in torch, in fp32 under autocast too (fp64 operands in fp64); rows without a pair are 0, whatever their
    operands hold.  ``dropout`` of the probabilities."""
    _check_operands(q, k, v, table, buckets)  # an index past the table would be read
    with torch.autocast(q.device.type, enabled=False):
        return _attention_torch(q, k, v, table, buckets, scale, dropout)


def _attention_torch(q, k, v, table, buckets: PairBuckets, scale: float, dropout: float):
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    allowed = buckets.allowed()
    has_key, has_query = allowed.any(2)[:, None, :, None], allowed.any(1)[:, None, :, None]
    none = torch.zeros((), dtype=q.dtype, device=q.device)
    q, k, v = torch.where(has_key, q, none), torch.where(has_query, k, none), torch.where(has_query, v, none)
    group = q.shape[1] // k.shape[1] if k.shape[1] else 1
    k, v = (t.to(wide).repeat_interleave(group, dim=1) for t in (k, v))
    bias = table_with_masked(table.to(wide))[table_rows(buckets)].permute(0, 3, 1, 2)
    s = torch.matmul(q.to(wide), k.transpose(-1, -2).contiguous()) * scale + bias
    if s.shape[-1] == 0:  # no maximum; zeros with gradients of zeros
        return torch.matmul(s, v).to(q.dtype), s.sum(-1).to(torch.float32)
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    some = total > 0
    p = p / torch.where(some, total, torch.ones_like(total))
    out = torch.matmul(torch.nn.functional.dropout(p, dropout) if dropout > 0.0 else p, v)
    out = torch.where(has_key, out, torch.zeros_like(out))
    lse = torch.where(some, torch.log(torch.where(some, total, torch.ones_like(total))) + top, torch.zeros_like(top))
    return out.to(q.dtype), lse[..., 0].to(torch.float32)


def bucket_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, buckets: PairBuckets, *,
                     scale: float | None = None, return_lse: bool = False):
    """softmax_j(scale q_i . k_j + table[bucket(i, j), h]) v_j over the keys j whose pair with i is not left out.

    q (B, H, Nq, D), k and v (B, KV, Nk, D), bf16 or fp16, D a multiple of 8 up to 128; KV divides H and each of its
    heads serves H / KV (at most 32) of q's.  They may be views, such as the heads of projected rows (entries of a head
    next to one another).  table (num_buckets, H) fp32, fp16 or bf16; its entries may be -inf.  ``buckets`` of a batch of B,
    or of one for every entry; scale D^-1/2 unless given.  One new token is Nq = 1.

    Returns out like q and, with return_lse, lse (B, H, Nq) fp32.  Queries without a pair get 0 (lse 0); keys and
    queries without a pair may hold anything (NaN); a key that some query attends must be finite.  Differentiable in q,
    k, v and the table through out and lse, for which the buckets need their transpose (made with gradients=True); two
    calls give identical bits."""
    _check_operands(q, k, v, table, buckets)
    B, H, Nq, D = q.shape
    KV, Nk = k.shape[1:3]
    s = float(D ** -0.5 if scale is None else scale) if D else 1.0
    if not math.isfinite(s):
        raise ValueError("scale must be finite")
    if q.device.type != "cuda":
        out, lse = bucket_attention_torch(q, k, v, table, buckets, s)
        return (out, lse) if return_lse else out
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("bucket_attention only supports float16/bfloat16 q, k, v of one dtype")
    if table.dtype not in _TABLE_DTYPES:
        raise RuntimeError(f"bucket_attention only supports a float32/float16/bfloat16 table, got {table.dtype}")
    if D < 8 or D > 128 or D % 8:
        raise RuntimeError(f"bucket_attention supports head_dim multiples of 8 up to 128, got {D}")
    if KV and H // KV > 32:
        raise RuntimeError(f"bucket_attention supports up to 32 heads to a key head, got {H // KV}")
    if any(n >= 1 << 31 for n in (B, H, Nq, Nk)):  # before they are cut to 32 bits
        raise RuntimeError(f"bucket_attention supports counts below 2^31, got {(B, H, Nq, Nk)}")
    check_layout(buckets)
    qo, ko, vo, t = _operand(q), _operand(k), _operand(v), table.contiguous()
    if _native.takes_gradient(q, k, v, table):
        if buckets.index_t is None:
            raise ValueError("gradients need buckets made with gradients=True")
        out, lse = _BucketAttentionFunction.apply(qo, ko, vo, t, buckets, s)
    else:
        out, lse, *_ = _forward(qo, ko, vo, t, buckets, s, lse=return_lse, training=False)
    return (out, lse) if return_lse else out
