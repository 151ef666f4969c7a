"""mf_gated_linear and mf_gated_linear_bwd against float64, element by element.

Tolerances, from the arithmetic.  u = 2^-24.  A sum of n products in fp32, in any order, is within n u sum|x w| of the
exact one (n products and n - 1 additions; the matrix cores add exactly or in fp32); with the bias one more.  So a and
b are within ea = (C + 1) u (|x| |Wg|^T + |bg|) and eb alike.  The activations have |act'| <= 1.13 (gelu) and
|act''| <= 0.8; evaluated in fp32 they are off by a few u (16-bit types: a few units of hardware exp2 and reciprocal and
the rounding of the exponent, below |x| u per exponent: 64 u covers |a| <= 30, where the inputs here lie; fp32: 16 u).
With y = act(a):
  |dh| <= 1.13 ea |b| + |y| eb + k u (|y b|)                                    k = 64 or 16
  |dA - exact| <= |go| (1.13 eb + 0.8 ea |b| + k u |b act'| + k u |b|),  |dB - exact| <= |go| (1.13 ea + k u |y| + k u)
and dA, dB are rounded to the type (eps / 2 relative) before the two products, which add their own fp32 sums: with
E = the error of [dA dB] just named,
  |dx - exact| <= E |W| + (2F + 1) u |[dA dB]| |W|,   |dW - exact| <= E^T |x| + (T + 1) u |[dA dB]|^T |x|.
dbias sums the unrounded values.  Each output rounds once more, eps / 2 relative or half the smallest subnormal."""

import math

import pytest
import torch

from matterformer_amd.gated_mlp import ACTIVATIONS, gated_linear

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def _act64(a, name):
    """Value and derivative in float64."""
    sig = torch.sigmoid(a)
    if name == "relu":
        return a.clamp_min(0), (a > 0).double()
    if name == "sigmoid":
        return sig, sig * (1 - sig)
    if name == "silu":
        return a * sig, sig * (1 + a * (1 - sig))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-a / math.sqrt(2.0))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(c * (a + 0.044715 * a ** 3))
    return a * s, s + a * s * (1 - s) * c * (1 + 3 * 0.044715 * a * a)


def _inputs(T, C, F, dtype, bias, seed, device, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, C, generator=gen) * scale).to(dtype)
    w = ((torch.rand(2 * F, C, generator=gen) * 2 - 1) * C ** -0.5).to(dtype)
    b = (torch.rand(2 * F, generator=gen) - 0.5).to(dtype) if bias else None
    go = (torch.randn(T, F, generator=gen) * 0.1).to(dtype)
    return [None if t is None else t.to(device) for t in (x, w, b, go)]


def _reference(x, w, b, go, name):
    """Outputs in float64 and their bounds before the last rounding."""
    x, w, go = x.double(), w.double(), go.double()
    C, F, T = x.shape[1], w.shape[0] // 2, x.shape[0]
    b = torch.zeros(2 * F, dtype=torch.float64, device=x.device) if b is None else b.double()
    both = x @ w.T + b
    e = (C + 1) * U * (x.abs() @ w.abs().T + b.abs())
    (a, up), (ea, eb) = both.chunk(2, -1), e.chunk(2, -1)
    y, dy = _act64(a, name)
    return x, w, go, a, up, ea, eb, y, dy, C, F, T


def _close(got, want, bound, what):
    fi = torch.finfo(got.dtype)
    tol = bound + (want.abs() + bound) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    err = (got.double() - want).abs()
    over = err - tol
    assert torch.all(over <= 0), f"{what}: off by {float(err.max()):.3e}, {float(over.max()):.3e} past the bound"


def _check(x, w, b, go, name, got, grads=None):
    dtype = x.dtype
    k = 16 if dtype == torch.float32 else 64
    half = torch.finfo(dtype).eps / 2
    X, W, GO, a, up, ea, eb, y, dy, C, F, T = _reference(x, w, b, go, name)
    _close(got, y * up, 1.13 * ea * up.abs() + y.abs() * eb + k * U * (y * up).abs(), "h")
    if grads is None:
        return
    da, db = GO * up * dy, GO * y
    fa = GO.abs() * (1.13 * eb + 0.8 * ea * up.abs() + k * U * (up * dy).abs() + k * U * up.abs())
    fb = GO.abs() * (1.13 * ea + k * U * y.abs() + k * U)
    dab, fab = torch.cat([da, db], -1), torch.cat([fa, fb], -1)
    tiny = torch.finfo(dtype).smallest_normal * half
    rounded = fab + (dab.abs() + fab) * half + tiny
    dx, dw, dbias = grads
    mag = dab.abs() + rounded
    _close(dx, dab @ W, rounded @ W.abs() + (2 * F + 1) * U * (mag @ W.abs()), "dx")
    _close(dw, dab.T @ X, rounded.T @ X.abs() + (T + 1) * U * (mag.T @ X.abs()), "dW")
    if b is not None:
        _close(dbias, dab.sum(0), fab.sum(0) + (T + 1) * U * (dab.abs() + fab).sum(0), "dbias")


def _run(x, w, b, go, name):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    out = gated_linear(*leaves, activation=name)
    grads = torch.autograd.grad(out, leaves, go)
    return out.detach(), [*grads, *([None] if b is None else [])]


SIZES = [
    # T, C, F
    (1, 8, 1), (1, 512, 256), (3, 17, 5), (16, 64, 64), (17, 72, 65), (33, 200, 100), (64, 128, 129), (65, 63, 200),
    (129, 136, 64), (300, 512, 341), (1000, 96, 128), (257, 1000, 70),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,C,F", SIZES)
def test_sizes(cuda, dtype, T, C, F):
    print(f"gated T={T} C={C} F={F} {dtype}", flush=True)
    x, w, b, go = _inputs(T, C, F, dtype, (T + C) % 2 == 0, T * 7 + C, cuda)
    out, grads = _run(x, w, b, go, "silu")
    _check(x, w, b, go, "silu", out, grads)
    with torch.no_grad():
        again = gated_linear(x, w, b)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_activations(cuda, dtype, activation):
    x, w, b, go = _inputs(130, 96, 80, dtype, True, 5, cuda, scale=4.0)
    _check(x, w, b, go, activation, *_run(x, w, b, go, activation))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_tiles(cuda, dtype):
    """Enough tiles of 256 for every CU in each of the three products, rows and columns that end inside one."""
    T, C, F = (4000, 1096, 1025) if dtype == torch.bfloat16 else (4000, 1096, 1025)
    x, w, b, go = _inputs(T, C, F, dtype, True, 11, cuda)
    _check(x, w, b, go, "gelu_tanh", *_run(x, w, b, go, "gelu_tanh"))


@pytest.mark.parametrize("dtype", TYPES)
def test_two_calls_give_identical_bits(cuda, dtype):
    x, w, b, go = _inputs(700, 256, 192, dtype, True, 12, cuda)
    one, two = _run(x, w, b, go, "silu"), _run(x, w, b, go, "silu")
    assert torch.equal(one[0], two[0]) and all(torch.equal(p, q) for p, q in zip(one[1], two[1]))


def test_views(cuda):
    """Rows apart (a slice of wider rows), more leading axes, a transposed weight, an expanded gradient."""
    x, w, b, go = _inputs(60, 80, 48, torch.bfloat16, True, 13, cuda)
    wide = torch.full((60, 120), float("nan"), dtype=torch.bfloat16, device=cuda)
    for start in (0, 8, 3):  # aligned twice, then not
        part = wide[:, start:start + 80]
        part.copy_(x)
        assert torch.equal(gated_linear(part, w, b), gated_linear(x, w, b))
    assert torch.equal(gated_linear(x.view(3, 4, 5, 80), w, b).view(60, 48), gated_linear(x, w, b))
    assert torch.equal(gated_linear(x, w.t().contiguous().t(), b), gated_linear(x, w, b))
    assert torch.equal(gated_linear(x[0], w, b), gated_linear(x[:1], w, b)[0])
    one = x[:1].expand(60, 80)
    assert torch.equal(gated_linear(one, w, b), gated_linear(one.contiguous(), w, b))
    leaf = x.clone().requires_grad_(True)
    gated_linear(leaf, w, b).sum().backward()
    _check(x, w, b, torch.ones_like(go), "silu", gated_linear(x, w, b),
           [leaf.grad, *_run(x, w, b, torch.ones_like(go), "silu")[1][1:]])


def test_gradients_of_some_inputs(cuda):
    x, w, b, go = _inputs(40, 64, 32, torch.bfloat16, True, 14, cuda)
    _, full = _run(x, w, b, go, "silu")
    for needs in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, w, b), needs)]
        grads = torch.autograd.grad(gated_linear(*leaves), [t for t, n in zip(leaves, needs) if n], go)
        assert all(torch.equal(g, f) for g, f in zip(grads, [f for f, n in zip(full, needs) if n]))


def test_gradient_against_differences(cuda):
    x, w, b, go = _inputs(9, 24, 12, torch.float32, True, 15, cuda)
    _, grads = _run(x, w, b, go, "gelu")
    gen = torch.Generator().manual_seed(16)
    for leaf, grad in zip((x, w, b), grads):
        step = torch.randn(leaf.shape, generator=gen).to(cuda)
        ends = []
        for s in (1.0, -1.0):
            t = [v.double() for v in (x, w, b)]
            t = [v + s * 1e-4 * step.double() if v.shape == leaf.shape else v for v in t]
            both = t[0] @ t[1].T + t[2]
            ends.append(float((_act64(both[:, :12], "gelu")[0] * both[:, 12:] * go.double()).sum()))
        slope = float((grad.double() * step.double()).sum())
        size = float((grad.double() * step.double()).abs().sum())
        # central differences of step 1e-4 in float64: third derivatives of order 10 leave 1e-8 relative to the sum;
        # the gradient's own sums carry about 60 roundings
        assert abs((ends[0] - ends[1]) / 2e-4 - slope) <= size * 200 * U + 1e-6


def test_rows_of_other_tokens_stay_apart(cuda):
    """NaN and infinity in one token's row reach that row only (and every weight gradient)."""
    x, w, b, go = _inputs(130, 64, 70, torch.bfloat16, True, 17, cuda)
    bad = x.clone()
    bad[129, 3] = float("nan")
    bad[5, 7] = float("inf")
    out, (dx, _, _) = _run(bad, w, b, go, "silu")
    ref, (rx, _, _) = _run(x, w, b, go, "silu")
    keep = torch.ones(130, dtype=torch.bool, device=cuda)
    keep[[5, 129]] = False
    assert torch.equal(out[keep], ref[keep]) and torch.equal(dx[keep], rx[keep])
    assert torch.isnan(out[129]).all()


def test_empty(cuda):
    w = torch.zeros(8, 16, device=cuda, requires_grad=True)
    b = torch.zeros(8, device=cuda, requires_grad=True)
    x = torch.zeros(0, 16, device=cuda, requires_grad=True)
    out = gated_linear(x, w, b)
    assert out.shape == (0, 4)
    dx, dw, db = torch.autograd.grad(out, (x, w, b), torch.zeros(0, 4, device=cuda))
    assert dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


def test_gpu_refusals(cuda):
    with pytest.raises(RuntimeError, match="bfloat16, float16 and float32"):
        gated_linear(torch.zeros(2, 8, device=cuda).double(), torch.zeros(4, 8, device=cuda).double())
    with pytest.raises(RuntimeError, match="share a dtype and a device"):
        gated_linear(torch.zeros(2, 8, device=cuda), torch.zeros(4, 8))


@pytest.mark.parametrize("C", [128, 100, 77])
def test_stream_and_graph(cuda, C):
    """Forward and backward on a side stream, then captured and replayed with eager work in between; with C = 77 the
    aligned copies are part of the graph."""
    x, w, b, go = _inputs(300, C, 96, torch.bfloat16, True, 18, cuda)
    want = _run(x, w, b, go, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(x, w, b, go, "silu")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _run(x, w, b, go, "silu")
    gen = torch.Generator().manual_seed(19)
    for turn in range(3):
        x.copy_(torch.randn(300, C, generator=gen).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        now = _run(x, w, b, go, "silu")
        assert torch.equal(held[0], now[0]) and all(torch.equal(p, q) for p, q in zip(held[1], now[1])), turn


def test_many_rows_pass_32_bit_offsets(cuda):
    """1.1e6 rows of 2048 hidden columns: 2.25e9 output elements; the last rows against a call of their own."""
    x, w, b, _ = _inputs(1100000, 64, 2048, torch.bfloat16, True, 20, cuda)
    with torch.no_grad():
        out = gated_linear(x, w, b)
        tail = gated_linear(x[-512:], w, b)
    assert torch.equal(out[-512:], tail)


def test_two_calls_in_flight(cuda):
    x, w, b, go = _inputs(70, 64, 40, torch.bfloat16, True, 21, cuda)
    leaf = x.clone().requires_grad_(True)
    one, two = gated_linear(leaf, w, b), gated_linear(leaf, w, b, activation="relu")
    g2 = torch.autograd.grad(two, leaf, go)[0]
    g1 = torch.autograd.grad(one, leaf, go)[0]
    assert torch.equal(g1, _run(x, w, b, go, "silu")[1][0]) and torch.equal(g2, _run(x, w, b, go, "relu")[1][0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [2047, 2305])
def test_either_side_of_the_tile_rule(cuda, dtype, T):
    """Half as many large tiles as CUs and a few more, rows that end inside a tile."""
    x, w, b, go = _inputs(T, 72, 2040, dtype, True, 22, cuda)
    _check(x, w, b, go, "silu", *_run(x, w, b, go, "silu"))


def test_aligned_copy_of_2_32_elements(cuda):
    """Rows of 255 channels are copied into rows of 256: 2^32 + 2^14 elements, more than a launch has threads."""
    x = torch.empty(2 ** 24 + 64, 255, dtype=torch.bfloat16, device=cuda).normal_()
    _, w, b, _ = _inputs(1, 255, 4, torch.bfloat16, True, 23, cuda)
    with torch.no_grad():
        out = gated_linear(x, w, b)
    for rows in (slice(0, 128), slice(2 ** 24 - 64, 2 ** 24 + 64)):
        _check(x[rows], w, b, x[rows, :4], "silu", out[rows])


def test_c_entries_refuse_a_workspace_off_16_bytes(cuda):
    from matterformer_amd import _native

    x, w, _, go = _inputs(4, 63, 32, torch.bfloat16, False, 24, cuda)
    out, work = torch.zeros(4, 32, dtype=x.dtype, device=cuda), torch.zeros(1 << 20, dtype=torch.uint8, device=cuda)
    a = _native.MfGatedLinearArgs(x=x.data_ptr(), weight=w.data_ptr(), out=out.data_ptr(), workspace=work.data_ptr() + 8,
                                  workspace_bytes=work.numel() - 8, x_stride=63, tokens=4, channels=63, hidden=32,
                                  dtype=_native.MF_DTYPE_BF16)
    b = _native.MfGatedLinearBwdArgs(fwd=a, grad_out=go.data_ptr(), dx=x.data_ptr(), workspace=work.data_ptr() + 8,
                                     workspace_bytes=work.numel() - 8)
    for name, args in (("mf_gated_linear", a), ("mf_gated_linear_bwd", b)):
        assert getattr(_native.lib(), name)(args, None) == _native.MF_ERR_INVALID_ARGUMENT
        assert "16-byte aligned" in _native.last_error()
    assert not out.any() and not work.any()


# float16's [dA dB] is kept times a power of two per token, chosen from the bound
#   B_n = 1.25 max|go_n| max(|x_n| max|Wu| + max|bu|, |x_n| max|Wg| + max|bg|, 1)     (Euclidean norms of rows)
# so that B_n 2^e_n lies in [2^13, 2^14): no value overflows, and what rounding leaves below the normal numbers, 2^-25
# 2^-e_n, is at most 2^-38 B_n.  For dW the rows come to the smallest e of all: the same with max B, once more rounded.
def _half_check(x, w, b, go, name, grads):
    X, W, GO, a, up, ea, eb, y, dy, C, F, T = _reference(x, w, b, go, name)
    t = 2.0 ** -11
    da, db = GO * up * dy, GO * y
    fa = GO.abs() * (1.13 * eb + 0.8 * ea * up.abs() + 64 * U * (up * dy).abs() + 64 * U * up.abs())
    fb = GO.abs() * (1.13 * ea + 64 * U * y.abs() + 64 * U)
    dab, fab = torch.cat([da, db], -1), torch.cat([fa, fb], -1)
    norm, size = X.norm(dim=1, keepdim=True), W.norm(dim=1)
    bias = torch.zeros(2 * F, dtype=torch.float64, device=x.device) if b is None else b.double().abs()
    reach = [norm * size[h].max() + bias[h].max() for h in (slice(0, F), slice(F, None))]
    bound = 1.25 * GO.abs().amax(1, keepdim=True) * torch.maximum(*reach).clamp_min(1.0)
    rounded = fab + (dab.abs() + fab) * t
    by_row = rounded + 2.0 ** -38 * bound
    by_all = rounded + 2.0 ** -37 * bound.max()
    for got, want, slack, what in (
            (grads[0], dab @ W, by_row @ W.abs() + (2 * F + 1) * U * ((dab.abs() + by_row) @ W.abs()), "dx"),
            (grads[1], dab.T @ X, by_all.T @ X.abs() + (T + 1) * U * ((dab.abs() + by_all).T @ X.abs()), "dW")):
        # a value past float16's range rounds to infinity (65520 and more), one within its bound of that may
        over, near = want.abs() - slack * (1 + t) >= 65520, want.abs() + slack * (1 + t) >= 65504
        assert torch.equal(got[over].double(), torch.sign(want[over]) * math.inf), what
        _close(torch.where(near, 0, got), torch.where(near, 0.0, want), torch.where(near, 0.0, slack), what)


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("T,C,F", [(40, 64, 48), (150, 80, 70)])
@pytest.mark.parametrize("sizes", [(30.0, 0.02, 3e4), (0.02, 30.0, 3e4), (0.02, 30.0, 1e-6), (1.0, 1.0, 1e-6)])
def test_half_gradients_near_the_ends_of_the_type(cuda, activation, T, C, F, sizes):
    """Intermediate gradients of 1e5 (past float16's largest number) and of 1e-6 (below its normal ones) whose dx or dW
    is within it."""
    gen = torch.Generator().manual_seed(T)
    x, w, go = (((torch.rand(*s, generator=gen) * 2 - 1) * m).half().to(cuda)
                for s, m in zip(((T, C), (2 * F, C), (T, F)), sizes))
    out, grads = _run(x, w, None, go, activation)
    assert torch.isfinite(out).all()
    X, W, GO, a, up, _, _, y, dy, *_ = _reference(x, w, None, go, activation)
    if sizes[2] > 1:
        assert float(torch.maximum((GO * up * dy).abs().max(), (GO * y).abs().max())) > 65504 or activation == "sigmoid"
    _half_check(x, w, None, go, activation, grads)


@pytest.mark.parametrize("T", [40, 300, 2500])
def test_half_gradients_of_other_tokens_stay_apart(cuda, T):
    """One token of 6e4 (its gradients overflow) changes no other token's dx; dW follows its formula with a token of 1e3."""
    x, w, b, go = _inputs(T, 64, 520, torch.float16, True, 25, cuda)
    big_x, big_go = x.clone(), go.clone()
    big_x[7], big_go[7] = 6e4, 6e4
    ref, got = _run(x, w, b, go, "silu")[1], _run(big_x, w, b, big_go, "silu")[1]
    keep = torch.arange(T, device=cuda) != 7
    assert torch.equal(got[0][keep], ref[0][keep])
    x[7] *= 8
    go[7] *= 1e3
    _half_check(x, w, b, go, "silu", _run(x, w, b, go, "silu")[1])
    want = _run(x, w, b, go, "silu")[1][0]
    go[T - 1] = float("inf")  # nor does a token that is not finite
    assert torch.equal(_run(x, w, b, go, "silu")[1][0][:T - 1], want[:T - 1])


@pytest.mark.parametrize("C", [128, 77])
def test_half_gradients_in_a_graph(cuda, C):
    """The scales are found anew at every replay: inputs of other magnitudes, checked against eager calls."""
    x, w, b, go = _inputs(300, C, 96, torch.float16, True, 26, cuda)
    _run(x, w, b, go, "silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _run(x, w, b, go, "silu")
    gen = torch.Generator().manual_seed(27)
    for size in (1e-4, 1e3, 1.0, 1e-6):
        go.copy_((torch.randn(300, 96, generator=gen) * size).half())
        x.copy_(torch.randn(300, C, generator=gen).half())
        graph.replay()
        torch.cuda.synchronize()
        now = _run(x, w, b, go, "silu")
        assert torch.equal(held[0], now[0]) and all(torch.equal(p, q) for p, q in zip(held[1], now[1])), size
        _half_check(x, w, b, go, "silu", now[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_far_apart(cuda, dtype):
    """Rows 2^22 elements apart, past what a tile's offsets reach: copied, not refused."""
    x, w, b, go = _inputs(5, 64, 40, dtype, True, 28, cuda)
    wide = torch.zeros(5, 1 << 22, dtype=dtype, device=cuda)
    wide[:, :64] = x
    out, grads = _run(wide[:, :64], w, b, go, "silu")
    _check(x, w, b, go, "silu", out, grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,C,F", [(4100, 1096, 2047), (8200, 2104, 600)])
def test_large_tiles_of_both_gradients(cuda, dtype, T, C, F):
    """Sizes whose dx and dW are cut into tiles of 256 (tiles times pieces of 16 K steps reach the 256 CUs): 85 and 80
    tiles in three pieces each; 297 tiles, 256 whole and 41 in five pieces, and 45 tiles in five.  Every edge is ragged."""
    x, w, b, go = _inputs(T, C, F, dtype, True, 29, cuda)
    out, grads = _run(x, w, b, go, "silu")
    _check(x, w, b, go, "silu", out, grads)
    again = _run(x, w, b, go, "silu")[1]
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_past_2_31_intermediate_elements(cuda, dtype):
    """2^24 + 300 tokens of 2 x 64 intermediate values: dx of the first and last tokens, and dW, to which only those
    contribute (x is zero between them)."""
    T = 2 ** 24 + 300
    _, w, _, _ = _inputs(1, 8, 64, dtype, False, 30, cuda)
    gen = torch.Generator().manual_seed(31)
    x = torch.zeros(T, 8, dtype=dtype, device=cuda)
    rows = torch.cat([torch.arange(200), torch.arange(T - 400, T)]).to(cuda)
    x[rows] = torch.randn(600, 8, generator=gen).to(dtype).to(cuda)
    go = torch.empty(T, 64, dtype=dtype, device=cuda).normal_().mul_(0.1)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    out = gated_linear(*leaves)
    dx, dw = torch.autograd.grad(out, leaves, go)
    _check(x.detach()[rows], w.detach(), None, go[rows], "silu", out.detach()[rows], (dx[rows], dw, None))


def test_gelu_keeps_its_relative_accuracy_in_the_tail(cuda):
    """fp32, one channel, weights of one: h = gelu(a) a for a from -12 to 12.  The normal distribution comes within 10 units
    of 2^-24 (the fit 1, t, its last steps and the product 7, the exponential 2) and the three products that follow round
    once each: 16 units, relative also where gelu is 1e-32."""
    a = torch.cat([torch.linspace(-12.0, 12.0, 100001), torch.tensor([0.0, -1e-20, 1e-20])]).to(cuda)
    out = gated_linear(a[:, None], torch.ones(2, 1, device=cuda), activation="gelu")[:, 0]
    want = _act64(a.double(), "gelu")[0] * a.double()
    assert torch.all((out.double() - want).abs() <= 16 * U * want.abs() + 2.0 ** -126)
