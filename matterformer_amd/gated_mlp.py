"""The gated feed-forward block: h = act(x Wg^T + bg) * (x Wu^T + bu), then an output projection.

The reference's block is the ungated Mlp (src/matterformer/models/transformer.py:129-148); a gated one takes the place
of its fc1 and activation.  ``gated_linear`` is both projections, the activation and the product in one kernel
(csrc/gated.hip, mf_gated_linear) with gradients of x, weight and bias (mf_gated_linear_bwd, which forms the two
projections again instead of keeping them).  GPU tensors in bfloat16, float16 or float32 run the kernels; a missing
library raises.  CPU tensors take the torch formulation.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd.function import once_differentiable

from matterformer_amd import _native

ACTIVATIONS = tuple(_native.MF_ACT)

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_TORCH_ACT = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu,
              "sigmoid": torch.sigmoid}


def _arguments(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, activation: str,
               out: torch.Tensor | None) -> _native.MfGatedLinearArgs:
    if x.shape[0] > 1 << 30 or weight.numel() >= 1 << 31:  # before they are cut to 32 bits
        raise RuntimeError(f"gated_linear supports up to 2^30 tokens and weights below 2^31 bytes, got {x.shape[0]} tokens "
                           f"and a weight of {tuple(weight.shape)}")
    return _native.MfGatedLinearArgs(
        x=x.data_ptr(), weight=weight.data_ptr(), bias=_native.ptr(bias), out=_native.ptr(out),
        x_stride=x.stride(0) if x.shape[0] > 1 else x.shape[1], tokens=x.shape[0], channels=x.shape[1],
        hidden=weight.shape[0] // 2, activation=_native.MF_ACT[activation], dtype=_native.dtype_code(x.dtype))


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Rows as the kernels take them: copied unless their entries lie side by side and the rows apart, but not so far
    that a tile of 256 reaches 2^31 bytes."""
    apart = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    if x.stride(-1) != 1 or apart < x.shape[1] or apart * 256 * x.element_size() >= 1 << 31:
        return x.contiguous()
    return x


def _scratch(nbytes: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, activation: str) -> torch.Tensor:
    out = torch.empty(x.shape[0], weight.shape[0] // 2, dtype=x.dtype, device=x.device)
    if out.numel() == 0:
        return out
    lib = _native.lib()
    args = _arguments(x, weight, bias, activation, out)
    nbytes = int(lib.mf_gated_linear_workspace_size(args))
    scratch = _scratch(nbytes, x.device)
    args.workspace, args.workspace_bytes = _native.ptr(scratch), nbytes
    _native.launch("mf_gated_linear", args, x.device)
    return out


class _GatedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation):
        ctx.save_for_backward(x, weight, bias)
        ctx.activation = activation
        return _forward(x, weight, bias, activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        grad = grad.contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = torch.empty_like(bias) if bias is not None and need[2] else None
        if x.shape[0] == 0:
            return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_(), None
        args = _native.MfGatedLinearBwdArgs(
            fwd=_arguments(x, weight, bias, ctx.activation, None), grad_out=grad.data_ptr(), dx=_native.ptr(dx),
            dweight=_native.ptr(dw), dbias=_native.ptr(db))
        nbytes = int(_native.lib().mf_gated_linear_bwd_workspace_size(args))
        scratch = _scratch(nbytes, x.device)
        args.workspace, args.workspace_bytes = _native.ptr(scratch), nbytes
        _native.launch("mf_gated_linear_bwd", args, x.device)
        return dx, dw, db, None


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 activation: str = "silu") -> torch.Tensor:
    """act(x Wg^T + bg) * (x Wu^T + bu): x (..., C); weight (2F, C), Wg its first F rows and Wu its last; bias (2F,) or
    None; one dtype (under autocast, its dtype, unless they are float64).  ``activation``: silu, gelu, gelu_tanh, relu or
    sigmoid.  Returns (..., F), differentiable in x, weight and bias.  Sums, activation and product are fp32 on the GPU,
    rounded once.  Up to 2^30 tokens and weights below 2^31 bytes there; hidden below 2^21 (float32 2^20)."""
    if activation not in _native.MF_ACT:
        raise ValueError(f"Unsupported activation: {activation}; expected one of {ACTIVATIONS}")
    if weight.ndim != 2 or weight.shape[0] == 0 or weight.shape[0] % 2 != 0 or weight.shape[1] == 0:
        raise ValueError(f"weight must have shape (2 * hidden, channels), got {tuple(weight.shape)}")
    if x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must have shape (..., {weight.shape[1]}), got {tuple(x.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must have shape ({weight.shape[0]},), got {tuple(bias.shape)}")
    if torch.is_autocast_enabled(x.device.type):
        dtype = torch.get_autocast_dtype(x.device.type)
        x, weight, bias = (t if t is None or t.dtype == torch.float64 else t.to(dtype) for t in (x, weight, bias))
    if any(t is not None and (t.dtype != x.dtype or t.device != x.device) for t in (weight, bias)):
        raise RuntimeError("x, weight and bias must share a dtype and a device")
    if x.device.type != "cuda":
        gate, up = F.linear(x, weight, bias).chunk(2, dim=-1)
        return _TORCH_ACT[activation](gate) * up
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"gated_linear supports bfloat16, float16 and float32 on the GPU, got {x.dtype}")
    rows = _rows(x if x.ndim == 2 else x.reshape(-1, x.shape[-1]))
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if _native.takes_gradient(rows, weight, bias):
        out = _GatedLinearFunction.apply(rows, weight, bias, activation)
    else:
        out = _forward(rows, weight, bias, activation)
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], out.shape[-1])
