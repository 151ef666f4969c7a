"""mf_radius_attn_bwd on the CPU: the C entry's checks and its struct."""

import pytest
import torch

from matterformer_amd import _native
from matterformer_amd.geometry_ops import RadiusTables, _check_tables


def test_c_entry_refuses_before_any_device_call():
    lib = _native.lib()
    fake = 1 << 20  # never dereferenced: every call below fails validation first
    names = ("q", "k", "v", "out", "lse", "grad_out", "mask_bits", "mask_bits_t", "key_any", "query_any", "dq", "dk", "dv")

    def args(**kw):
        a = {n: fake for n in names}
        a.update(scale=0.125, batch=1, heads=1, atoms=4, head_dim=64, dtype=_native.MF_DTYPE_BF16)
        a.update(kw)
        return _native.MfRadiusAttnBwdArgs(**a)

    invalid, unsupported = _native.MF_ERR_INVALID_ARGUMENT, _native.MF_ERR_UNSUPPORTED
    assert lib.mf_radius_attn_bwd(None, None) == invalid and "args is NULL" in _native.last_error()
    for name in names:
        assert lib.mf_radius_attn_bwd(args(**{name: None}), None) == invalid and "non-NULL" in _native.last_error()
    for kw, status, match in ((dict(atoms=-1), invalid, "non-negative"), (dict(dtype=0), unsupported, "float16/bfloat16"),
                              (dict(head_dim=48), unsupported, "head_dim"),
                              (dict(scale=float("nan")), invalid, "finite"), (dict(dq=fake + 8), invalid, "aligned"),
                              (dict(atoms=65537), unsupported, "65536"), (dict(), invalid, "workspace"),
                              (dict(workspace=fake, workspace_bytes=64), invalid, "workspace")):
        assert lib.mf_radius_attn_bwd(args(**kw), None) == status
        assert match in _native.last_error()
    assert lib.mf_radius_attn_bwd(args(heads=0), None) == _native.MF_OK
    assert lib.mf_radius_attn_bwd_workspace_size(0, 1, 4, 2) == 0
    # fp16 keeps the peaks of every tile as well
    assert lib.mf_radius_attn_bwd_workspace_size(2, 3, 65, 1) > lib.mf_radius_attn_bwd_workspace_size(2, 3, 65, 2) > 0


def test_tables_entry_refuses_before_any_device_call():
    lib = _native.lib()
    fake = 1 << 20
    names = ("mask_bits", "mask_bits_t", "key_any", "query_any")

    def args(**kw):
        a = {n: fake for n in names}
        a.update(batch=1, atoms=4)
        a.update(kw)
        return _native.MfRadiusTablesArgs(**a)

    invalid = _native.MF_ERR_INVALID_ARGUMENT
    assert lib.mf_radius_tables(None, None) == invalid and "args is NULL" in _native.last_error()
    for name in names:
        assert lib.mf_radius_tables(args(**{name: None}), None) == invalid and "non-NULL" in _native.last_error()
    assert lib.mf_radius_tables(args(atoms=-1), None) == invalid
    assert lib.mf_radius_tables(args(atoms=65537), None) == _native.MF_ERR_UNSUPPORTED
    assert lib.mf_radius_tables(args(batch=0), None) == _native.MF_OK


def test_entries_refuse_more_threads_than_a_launch_has():
    lib = _native.lib()
    fake = 1 << 20
    names = ("q", "k", "v", "out", "lse", "grad_out", "mask_bits", "mask_bits_t", "key_any", "query_any", "dq", "dk", "dv",
             "workspace")
    a = _native.MfRadiusAttnBwdArgs(**{n: fake for n in names}, workspace_bytes=2 ** 60, scale=0.125, batch=2 ** 23, heads=1,
                                    atoms=1, head_dim=32, dtype=_native.MF_DTYPE_BF16)
    assert lib.mf_radius_attn_bwd(a, None) == _native.MF_ERR_UNSUPPORTED and "too large" in _native.last_error()
    t = _native.MfRadiusTablesArgs(**{n: fake for n in ("mask_bits", "mask_bits_t", "key_any", "query_any")}, batch=2 ** 26,
                                   atoms=1)
    assert lib.mf_radius_tables(t, None) == _native.MF_ERR_UNSUPPORTED and "too large" in _native.last_error()


def test_tables_of_another_form_are_refused():
    bits = torch.zeros(2, 70, 3, dtype=torch.int32)

    def tables(**kw):
        t = dict(bits_t=bits.clone(), key_any=torch.zeros(2, 2, 2, dtype=torch.int64),
                 query_any=torch.zeros(2, 2, 2, dtype=torch.int64))
        t.update(kw)
        return RadiusTables(**t)

    _check_tables(tables(), bits, (2, 2, 2))
    for kw in (dict(bits_t=bits[:1]), dict(bits_t=bits.long()), dict(key_any=torch.zeros(2, 1, 2, dtype=torch.int64)),
               dict(query_any=torch.zeros(2, 2, 1, dtype=torch.int64)), dict(query_any=torch.zeros(2, 2, 2)),
               dict(query_any=torch.zeros(2, 2, 2, dtype=torch.int64, device="meta")),
               dict(key_any=torch.zeros(2, 2, 2, dtype=torch.int64).transpose(0, 1))):
        with pytest.raises(ValueError, match="radius_tables of this call"):
            _check_tables(tables(**kw), bits, (2, 2, 2))
