"""Rotary positions on the CPU: the frequency table, the torch formulation, its gradients and the refusals."""

import math

import pytest
import torch

from matterformer_amd import _native
from matterformer_amd.rotary import RotaryFrequencies, apply_rotary, rotary_frequencies, rotary_heads
from rotary_reference import assert_turned, rotate64


def test_table_of_each_scaling():
    P, base, s, L = 8, 10000.0, 4.0, 4096.0
    plain = [base ** (-i / P) for i in range(P)]
    got = rotary_frequencies(16, base=base).table
    assert torch.allclose(got, torch.tensor(plain, dtype=torch.float64), rtol=1e-14, atol=0)
    got = rotary_frequencies(16, base=base, scaling="linear", factor=s).table
    assert torch.allclose(got, torch.tensor(plain, dtype=torch.float64) / s, rtol=1e-14, atol=0)
    got = rotary_frequencies(16, base=base, scaling="ntk", factor=s).table
    assert float(got[0]) == 1.0 and math.isclose(float(got[-1]), plain[-1] / s, rel_tol=1e-13)
    yarn = rotary_frequencies(16, base=base, scaling="yarn", factor=s, original_length=L)
    assert math.isclose(yarn.gain, 0.1 * math.log(s) + 1.0)
    for f, p in zip(yarn.table.tolist(), plain):
        turns = L * p / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
        assert math.isclose(f, keep * p + (1 - keep) * p / s, rel_tol=1e-13)
    assert float(yarn.table[0]) == 1.0 and math.isclose(float(yarn.table[-1]), plain[-1] / s, rel_tol=1e-13)


def test_axes_repeat_the_table():
    f = rotary_frequencies(24, axes=3, base=100.0)
    assert f.rotary_dim == 24 and f.axes == 3
    assert torch.equal(f.table[:4], f.table[4:8]) and torch.equal(f.table[:4], f.table[8:])


@pytest.mark.parametrize("kwargs,match", [
    (dict(rotary_dim=15), "multiple of 2"), (dict(rotary_dim=16, axes=3), "multiple of 6"),
    (dict(rotary_dim=16, axes=4), "axes"), (dict(rotary_dim=0), "positive"), (dict(rotary_dim=16, base=-1.0), "base"),
    (dict(rotary_dim=16, scaling="cubic"), "scaling"), (dict(rotary_dim=16, scaling="linear", factor=0.5), "factor"),
    (dict(rotary_dim=16, scaling="yarn", factor=2.0), "original_length"),
    (dict(rotary_dim=16, scaling="yarn", factor=2.0, original_length=64, beta_fast=1.0), "beta_fast")])
def test_frequency_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        rotary_frequencies(**kwargs)


def test_frequency_object_refusals():
    with pytest.raises(ValueError, match="float64"):
        RotaryFrequencies(torch.ones(4))
    with pytest.raises(ValueError, match="multiple of axes"):
        RotaryFrequencies(torch.ones(4, dtype=torch.float64), axes=3)
    with pytest.raises(ValueError, match="gain"):
        RotaryFrequencies(torch.ones(4, dtype=torch.float64), gain=float("nan"))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("R,axes", [(8, 1), (6, 3), (4, 2)])
def test_torch_formulation_and_gradient(layout, R, axes):
    gen = torch.Generator().manual_seed(R + axes)
    q = torch.randn(2, 3, 5, 8, generator=gen, dtype=torch.float64, requires_grad=True)
    k = torch.randn(2, 1, 5, 8, generator=gen, dtype=torch.float64, requires_grad=True)
    pos = torch.randn(2, 5, axes, generator=gen) * 10
    f = rotary_frequencies(R, axes=axes, base=50.0)
    out = apply_rotary(q, k, pos if axes > 1 else pos[..., 0], f, layout=layout)
    for x, y in zip((q, k), out):
        want, _ = rotate64(x, pos, f.table, axes, 1.0, layout)
        assert torch.allclose(y, want, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda a, b: apply_rotary(a, b, pos if axes > 1 else pos[..., 0], f, layout=layout),
                                    (q, k))


def test_products_depend_on_differences_only():
    gen = torch.Generator().manual_seed(3)
    q, k = (torch.randn(1, 2, 6, 12, generator=gen, dtype=torch.float64) for _ in range(2))
    pos = torch.randn(1, 6, 3, generator=gen, dtype=torch.float64)
    f = rotary_frequencies(12, axes=3, base=20.0)
    a, b = apply_rotary(q, k, pos, f)
    c, d = apply_rotary(q, k, pos + torch.tensor([1.5, -2.0, 0.25]), f)
    assert torch.allclose(a @ b.mT, c @ d.mT, rtol=1e-11, atol=1e-11)


def test_rows_equal_heads():
    gen = torch.Generator().manual_seed(4)
    rows = torch.randn(2, 7, (4 + 2) * 10, generator=gen)
    pos = torch.arange(7)[None]
    f = rotary_frequencies(8)
    q, k, v = rotary_heads(rows, pos, f, heads=4, kv_heads=1, layout="interleaved")
    hq, hk, hv = rows.split((40, 10, 10), dim=-1)
    a, b = apply_rotary(hq.view(2, 7, 4, 10).transpose(1, 2), hk.view(2, 7, 1, 10).transpose(1, 2),
                        pos.expand(2, 7), f, layout="interleaved")
    assert torch.equal(q, a) and torch.equal(k, b) and torch.equal(v, hv.view(2, 7, 1, 10).transpose(1, 2))
    assert all(t.is_contiguous() for t in (q, k, v))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_heads_in_another_dtype(layout):
    """Rounded once, from the rows' own type; the gradient comes in theirs."""
    gen = torch.Generator().manual_seed(5)
    rows = torch.randn(2, 7, 3 * 2 * 10, generator=gen, requires_grad=True)
    pos, f = torch.arange(7)[None] * 3, rotary_frequencies(8)
    q, k, v = rotary_heads(rows, pos, f, heads=2, layout=layout, dtype=torch.bfloat16)
    assert all(t.dtype == torch.bfloat16 for t in (q, k, v))
    for got, part in zip((q, k), rows.split(20, dim=-1)):
        part = part.reshape(2, 7, 2, 10).transpose(1, 2)
        assert_turned(got, *rotate64(part, pos.expand(2, 7), f.table, 1, 1.0, layout), layout)
    assert torch.equal(v, rows[..., 40:].reshape(2, 7, 2, 10).transpose(1, 2).bfloat16())
    (g,) = torch.autograd.grad((q, k, v), rows, [torch.ones_like(t) for t in (q, k, v)])
    assert g.dtype == torch.float32
    with pytest.raises(RuntimeError, match="heads"):
        rotary_heads(rows, pos, f, heads=2, dtype=torch.int32)


def test_argument_refusals():
    q = torch.zeros(2, 3, 5, 8)
    f = rotary_frequencies(8)
    pos = torch.zeros(2, 5)
    with pytest.raises(ValueError, match="layout"):
        apply_rotary(q, None, pos, f, layout="pairs")
    with pytest.raises(ValueError, match="greater than head_dim"):
        apply_rotary(q, None, pos, rotary_frequencies(16))
    with pytest.raises(ValueError, match="positions must have shape"):
        apply_rotary(q, None, torch.zeros(2, 4), f)
    with pytest.raises(ValueError, match="positions must have shape"):
        apply_rotary(q, None, torch.zeros(3, 5), f)
    with pytest.raises(ValueError, match="positions must have shape"):
        apply_rotary(q, None, torch.zeros(2, 5, 2), f)
    with pytest.raises(RuntimeError, match="must be float32"):
        apply_rotary(q, None, torch.zeros(2, 5, dtype=torch.float16), f)
    with pytest.raises(RuntimeError, match="no gradient"):
        apply_rotary(q, None, torch.zeros(2, 5, requires_grad=True), f)
    with pytest.raises(RuntimeError, match="share a dtype"):
        apply_rotary(q, q.double(), pos, f)
    with pytest.raises(ValueError, match="q must have shape"):
        apply_rotary(q, torch.zeros(2, 3, 4, 8), pos, f)
    with pytest.raises(ValueError, match="rows must have shape"):
        rotary_heads(torch.zeros(2, 5, 50), pos, f, heads=4)
    with pytest.raises(ValueError, match="positive"):
        rotary_heads(torch.zeros(2, 5, 48), pos, f, heads=4, kv_heads=0)


def test_a_table_that_asks_for_a_gradient_is_refused():
    f = RotaryFrequencies(torch.ones(4, dtype=torch.float64, requires_grad=True))
    for call in (lambda: apply_rotary(torch.zeros(1, 1, 5, 8), None, torch.zeros(1, 5), f),
                 lambda: rotary_heads(torch.zeros(1, 5, 24), torch.zeros(1, 5), f, heads=1)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()


def test_c_entry_refuses_before_any_device_call():
    lib = _native.lib()
    fake = 1 << 20  # never dereferenced: every call below fails validation first

    def args(**kw):
        a = _native.MfRotaryArgs(positions=fake, frequencies=fake, gain=1.0, parts=1, batch=1, tokens=4, head_dim=8,
                                 rotary_dim=8, axes=1, src_dtype=_native.MF_DTYPE_F32, dst_dtype=_native.MF_DTYPE_F32)
        a.src0 = a.dst0 = fake
        a.heads0 = 1
        for key, value in kw.items():
            setattr(a, key, value)
        return a

    assert lib.mf_rotary(None, None) == _native.MF_ERR_INVALID_ARGUMENT and "args is NULL" in _native.last_error()
    for kw, match in ((dict(parts=4), "parts"), (dict(positions=None), "non-NULL"), (dict(tokens=-1), "sizes"),
                      (dict(axes=4), "axes"), (dict(rotary_dim=7), "rotary_dim"), (dict(rotary_dim=10), "rotary_dim"),
                      (dict(src_dtype=9), "dtype"), (dict(position_type=4), "position_type"),
                      (dict(slot_side=1), "slot map"), (dict(slot_side=3), "slot_side"),
                      (dict(gain=float("inf")), "gain"), (dict(parts=2), "needs src and dst")):
        assert lib.mf_rotary(args(**kw), None) == _native.MF_ERR_INVALID_ARGUMENT
        assert match in _native.last_error()
    assert lib.mf_rotary(args(head_dim=264), None) == _native.MF_ERR_UNSUPPORTED
    bad = args()
    bad.src_stride0 = -8
    assert lib.mf_rotary(bad, None) == _native.MF_ERR_INVALID_ARGUMENT and "strides" in _native.last_error()
    assert lib.mf_rotary(args(tokens=0), None) == _native.MF_OK


def test_struct_has_the_header_layout(tmp_path):
    """The flat fields lie where the C compiler puts the arrays' elements."""
    import shutil
    import subprocess
    from pathlib import Path

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mf_capi.h"', "int main(void) {"]
    want = {}
    for name, *_ in _native.MfRotaryArgs._fields_:
        base = name.rstrip("0123456789")
        field = name
        if base != name:
            i = int(name[len(base):])
            field = f"{base}[{i // 3}][{i % 3}]" if base in ("src_stride", "dst_stride") else f"{base}[{i}]"
        lines.append(f'  printf("{name} %zu\\n", offsetof(mf_rotary_args, {field}));')
        want[name] = getattr(_native.MfRotaryArgs, name).offset
    lines += ['  printf("size %zu\\n", sizeof(mf_rotary_args));', "  return 0;", "}"]
    (tmp_path / "t.c").write_text("\n".join(lines))
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, f"-I{include}", str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout
    got = {line.split()[0]: int(line.split()[1]) for line in out.splitlines()}
    import ctypes

    assert got.pop("size") == ctypes.sizeof(_native.MfRotaryArgs)
    assert got == want


@pytest.mark.parametrize("name,argtype", [("mf_radius_attn_args", _native.MfRadiusAttnArgs),
                                          ("mf_radius_tables_args", _native.MfRadiusTablesArgs),
                                          ("mf_radius_attn_bwd_args", _native.MfRadiusAttnBwdArgs),
                                          ("mf_gated_linear_args", _native.MfGatedLinearArgs),
                                          ("mf_gated_linear_bwd_args", _native.MfGatedLinearBwdArgs)])
def test_the_other_new_structs_have_the_header_layout(tmp_path, name, argtype):
    import ctypes
    import shutil
    import subprocess
    from pathlib import Path

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mf_capi.h"', "int main(void) {"]
    lines += [f'  printf("{f} %zu\\n", offsetof({name}, {f}));' for f, *_ in argtype._fields_]
    lines += [f'  printf("size %zu\\n", sizeof({name}));', "  return 0;", "}"]
    (tmp_path / "t.c").write_text("\n".join(lines))
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, f"-I{include}", str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout
    got = {line.split()[0]: int(line.split()[1]) for line in out.splitlines()}
    assert got.pop("size") == ctypes.sizeof(argtype)
    assert got == {f: getattr(argtype, f).offset for f, *_ in argtype._fields_}


def test_c_entry_refuses_more_threads_than_a_launch_has():
    fake = 1 << 20
    a = _native.MfRotaryArgs(positions=fake, frequencies=fake, gain=1.0, parts=1, batch=1, tokens=2 ** 28, head_dim=2,
                             rotary_dim=2, axes=1, src_dtype=_native.MF_DTYPE_BF16, dst_dtype=_native.MF_DTYPE_BF16)
    a.src0 = a.dst0 = fake
    a.heads0 = 1
    assert _native.lib().mf_rotary(a, None) == _native.MF_ERR_UNSUPPORTED and "too many tokens" in _native.last_error()
