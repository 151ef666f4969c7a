"""The gated linear layer on the CPU: the torch formulation, the refusals and the C entry's checks."""

import pytest
import torch

from matterformer_amd import _native
from matterformer_amd.gated_mlp import ACTIVATIONS, gated_linear


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("bias", [True, False])
def test_torch_formulation(activation, bias):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 5, generator=gen, dtype=torch.float64, requires_grad=True)
    w = torch.randn(8, 5, generator=gen, dtype=torch.float64, requires_grad=True)
    b = torch.randn(8, generator=gen, dtype=torch.float64, requires_grad=True) if bias else None
    act = {"silu": lambda a: a / (1 + torch.exp(-a)), "gelu": lambda a: a * 0.5 * (1 + torch.erf(a / 2 ** 0.5)),
           "gelu_tanh": lambda a: 0.5 * a * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (a + 0.044715 * a ** 3))),
           "relu": lambda a: a * (a > 0), "sigmoid": lambda a: 1 / (1 + torch.exp(-a))}[activation]
    both = x @ w.T + (b if bias else 0.0)
    got = gated_linear(x, w, b, activation=activation)
    assert got.shape == (2, 3, 4)
    assert torch.allclose(got, act(both[..., :4]) * both[..., 4:], rtol=1e-12, atol=1e-12)


def test_refusals():
    x, w = torch.zeros(3, 5), torch.zeros(8, 5)
    with pytest.raises(ValueError, match="activation"):
        gated_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="weight must have shape"):
        gated_linear(x, torch.zeros(7, 5))
    with pytest.raises(ValueError, match="weight must have shape"):
        gated_linear(torch.zeros(3, 0), torch.zeros(8, 0))
    with pytest.raises(ValueError, match="x must have shape"):
        gated_linear(torch.zeros(3, 4), w)
    with pytest.raises(ValueError, match="bias must have shape"):
        gated_linear(x, w, torch.zeros(4))
    with pytest.raises(RuntimeError, match="share a dtype"):
        gated_linear(x, w.double())


def test_c_entries_refuse_before_any_device_call():
    lib = _native.lib()
    fake = 1 << 20  # never dereferenced: every call below fails validation first
    invalid, unsupported = _native.MF_ERR_INVALID_ARGUMENT, _native.MF_ERR_UNSUPPORTED

    def args(**kw):
        a = dict(x=fake, weight=fake, out=fake, x_stride=64, tokens=4, channels=64, hidden=32, dtype=2)
        a.update(kw)
        return _native.MfGatedLinearArgs(**a)

    assert lib.mf_gated_linear(None, None) == invalid and "args is NULL" in _native.last_error()
    assert lib.mf_gated_linear_bwd(None, None) == invalid and "args is NULL" in _native.last_error()
    assert lib.mf_gated_linear_workspace_size(None) == 0 and lib.mf_gated_linear_bwd_workspace_size(None) == 0
    for kw, status, match in ((dict(x=None), invalid, "non-NULL"), (dict(out=None), invalid, "out must be"),
                              (dict(tokens=-1), invalid, "tokens"), (dict(channels=0), invalid, "channels"),
                              (dict(hidden=0), invalid, "hidden"), (dict(x_stride=60), invalid, "x_stride"),
                              (dict(dtype=7), invalid, "dtype"), (dict(activation=5), invalid, "activation"),
                              (dict(hidden=1 << 24, channels=64), unsupported, "2^31")):
        assert lib.mf_gated_linear(args(**kw), None) == status
        assert match in _native.last_error()
    assert lib.mf_gated_linear(args(tokens=0), None) == _native.MF_OK
    # aligned operands need no workspace, odd channels two copies
    assert lib.mf_gated_linear_workspace_size(args()) == 0
    assert lib.mf_gated_linear_workspace_size(args(channels=63)) == 512 + 64 * 64 * 2
    b = _native.MfGatedLinearBwdArgs(fwd=args(), grad_out=fake)
    assert lib.mf_gated_linear_bwd(b, None) == invalid and "nothing to compute" in _native.last_error()
    b.grad_out = None
    assert lib.mf_gated_linear_bwd(b, None) == invalid and "grad_out" in _native.last_error()


def test_c_entries_name_the_limit_that_a_call_passes():
    """Offsets within a tile are 32 bits: each limit with its size, which half as many elements of fp32 reach."""
    lib = _native.lib()
    fake = 1 << 20

    def refusal(**kw):
        a = dict(x=fake, weight=fake, out=fake, x_stride=64, tokens=4, channels=8, hidden=32, dtype=2)
        a.update(kw)
        a["x_stride"] = max(a["x_stride"], a["channels"])
        assert lib.mf_gated_linear(_native.MfGatedLinearArgs(**a), None) == _native.MF_ERR_UNSUPPORTED
        return _native.last_error()

    assert "tokens" in refusal(tokens=(1 << 30) + 1)
    assert "weight" in refusal(channels=16384, hidden=53248)
    for dtype, most in ((2, 1 << 22), (0, 1 << 21)):
        assert f"rows of x {most} elements apart" in refusal(x_stride=most, dtype=dtype)
        assert f"hidden above {most // 2 - 65}" in refusal(channels=1, hidden=most // 2 - 64, dtype=dtype)


def test_rows_far_apart_are_copied():
    from matterformer_amd.gated_mlp import _rows

    assert _rows(torch.zeros(8).expand(3, 8)).is_contiguous()  # rows on top of each other
    near = torch.zeros(2, 16)[:, :8]
    assert _rows(near) is near
    one = torch.empty(1, 8).as_strided((1, 8), (1 << 40, 1))
    assert _rows(one) is one  # one row's stride means nothing
    for dtype, most in ((torch.bfloat16, 1 << 22), (torch.float32, 1 << 21)):
        base = torch.zeros(most + 8, dtype=dtype)
        assert _rows(base.as_strided((2, 8), (most - 8, 1))).stride(0) == most - 8
        assert _rows(base.as_strided((2, 8), (most, 1))).is_contiguous()


def test_autocast_leaves_float64_alone():
    """As it does F.linear; other types come to its own."""
    x, w = torch.randn(3, 5, dtype=torch.float64), torch.randn(8, 5, dtype=torch.float64)
    want = gated_linear(x, w)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert torch.nn.functional.linear(x, w).dtype == torch.float64
        got = gated_linear(x, w)
        assert gated_linear(x.float(), w.float()).dtype == torch.bfloat16
    assert got.dtype == torch.float64 and torch.equal(got, want)
