"""Attention with a bias by buckets in 64 bits, with its gradients and the bounds that roundings leave."""

import math

import torch

MASKED = 64


def step(dtype):
    """Half a step of a type, relative: what one rounding can be off by."""
    return torch.finfo(dtype).eps / 2


def dense(index, table):
    """(B, H, Nq, Nk) fp64 bias, -inf at pairs that are left out."""
    t = torch.cat([table.double(), table.new_full((1, table.shape[1]), -math.inf).double()])
    rows = torch.where(index == MASKED, table.shape[0], index.long())
    return t[rows].permute(0, 3, 1, 2)


def clean(t, keep):
    """Rows that no pair uses as zeros: what they hold reaches nothing."""
    return torch.where(keep[:, None, :, None], t.double(), 0.0)


def attention(q, k, v, table, index, scale, go=None, glse=None):
    """A dict of out, lse, (with go) dq, dk, dv, dtable, and of each the bound on |kernel - it|.

    The kernel rounds P and dS to the operands' type for their products and every result once more; S, softmax, delta and
    sums are fp32, where |x| < 128 leaves P a relative error below 128 * 2^-24 * 4 = 2^-15 (and delta's from out's two
    parts, 2^-18, is within the same share of its terms).  delta = go . out has the error of out's rounded P, at most
    (u + f) |go| . (P |v|), in dq; for dk and dtable it is corrected.
    fp16's steps end at 2^-24: a result is off by up to 2^-25 besides; P by 2^-32 (it is kept times 2^7 over a sum of at
    least 1) and, for dv, 2^-37 (kept times 2^12); and dS, kept times 2^e >= 2^12 / (2 max|go| max|v| + max|dlse|), by
    2^-25 - e."""
    half = q.dtype == torch.float16
    grain = 2.0 ** -25 if half else 0.0
    B, H = q.shape[:2]
    G = H // k.shape[1]
    u, f = step(q.dtype), 2.0 ** -15
    allowed = (index != MASKED).expand(B, *index.shape[1:])
    index = index.expand(B, *index.shape[1:])
    q64 = clean(q, allowed.any(2))
    k64, v64 = (clean(t, allowed.any(1)).repeat_interleave(G, dim=1) for t in (k, v))
    s = q64 @ k64.transpose(-1, -2).contiguous() * scale + dense(index, table)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    P = torch.where(total > 0, e / torch.where(total > 0, total, 1.0), 0.0)
    out = P @ v64
    r = {"out": out, "lse": torch.where(total > 0, torch.log(total) + top, 0.0)[..., 0]}
    spread = P @ v64.abs()
    bound = {"out": u * out.abs() + (u + f) * spread + grain + 2.0 ** -7 * grain * v64.abs().sum(2, keepdim=True), "lse": 2.0 ** -15 + r["lse"].abs() * 2.0 ** -20}
    if go is None:
        return r, bound
    g64 = clean(go, allowed.any(2))
    delta = (g64 * out).sum(-1, keepdim=True)
    wide = (g64.abs() * (out.abs() + spread * (u + f))).sum(-1, keepdim=True)
    if glse is not None:
        delta = delta - glse.double()[..., None]
        wide = wide + glse.double().abs()[..., None]
    dP = g64 @ v64.transpose(-1, -2).contiguous()
    dS = P * (dP - delta)
    off = P * (g64.abs() @ v64.abs().transpose(-1, -2).contiguous() + wide) * f  # of dS, before it is rounded
    per_key = lambda t: t.unflatten(1, (-1, G)).sum(2)
    r["dq"] = scale * dS @ k64
    r["dk"] = per_key(scale * dS.transpose(-1, -2).contiguous() @ q64)
    r["dv"] = per_key(P.transpose(-1, -2).contiguous() @ g64)
    sums, most = (torch.stack([torch.where(index[:, None] == c, t, 0.0).sum((0, 2, 3)) for c in range(table.shape[0])])
                  for t in (dS, off))
    r["dtable"] = sums
    peak = 2.0 * g64.norm(dim=-1).max() * v64.norm(dim=-1).max() + (0.0 if glse is None else glse.double().abs().max())
    dS_off = dS.abs() * u + off + grain * peak * 2.0 ** -12
    scale = abs(scale)
    of_delta = (g64.abs() * spread).sum(-1, keepdim=True) * (u + f) * (P @ k64.abs())
    bound["dq"] = scale * (dS_off @ k64.abs() + of_delta) + u * r["dq"].abs() + grain
    bound["dk"] = per_key(scale * dS_off.transpose(-1, -2).contiguous() @ q64.abs()) + u * r["dk"].abs() + grain
    bound["dv"] = (per_key(((u + f) * P + grain * 2.0 ** -12).transpose(-1, -2).contiguous() @ g64.abs())
                   + u * r["dv"].abs() + grain)
    bound["dtable"] = most + step(table.dtype) * r["dtable"].abs()
    return r, bound


def check(got, r, bound, floor=0.0):
    """got: a dict of some of r's names."""
    for name, t in got.items():
        off = (t.double() - r[name]).abs()
        worst = (off - bound[name] - floor).max().item() if off.numel() else 0.0
        assert worst <= 0.0, f"{name}: off by {off.max().item():.3e}, {worst:.3e} past its bound"
