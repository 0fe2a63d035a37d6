"""The state-space block's operators without a GPU: what the C entries and the Python layer refuse, and the host helpers."""
import ctypes

import numpy as np
import pytest

from mDeepFRI import _hip, ssm

P = 1 << 32      # addresses that nothing reads: every check runs before the device is touched


def conv(**kw):
    a = ssm._Conv()
    a.rows.lengths, a.rows.row_off, a.rows.R, a.rows.B, a.rows.max_len = P, P, 100, 4, 30
    a.x, a.weight, a.out, a.ldx, a.ldo, a.channels, a.width, a.dtype = P, P, 2 * P, 64, 64, 64, 4, _hip.DT_F32
    return _set(a, kw), _hip.lib().mdf_causal_conv_dev, ()


def scan(**kw):
    a = ssm._Scan()
    a.rows.lengths, a.rows.row_off, a.rows.R, a.rows.B, a.rows.max_len = P, P, 100, 4, 30
    a.x, a.b, a.c, a.dt, a.a, a.y = P, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P
    a.ldx, a.ldb, a.ldc, a.lddt, a.ldy = 128, 16, 16, 4, 128
    a.heads, a.groups, a.head_dim, a.state_dim, a.dtype, a.dt_dtype = 4, 2, 32, 8, _hip.DT_BF16, _hip.DT_BF16
    return _set(a, kw), _hip.lib().mdf_selective_scan_dev, (None, 0)


def step(**kw):
    a = ssm._Step()
    a.xbc, a.dt, a.conv_weight, a.a, a.conv_state, a.state, a.y = P, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P, 7 * P
    a.ldx, a.lddt, a.ldy, a.B, a.n_slots = 160, 4, 128, 3, 3
    a.heads, a.groups, a.head_dim, a.state_dim, a.width, a.dtype, a.dt_dtype = 4, 2, 32, 8, 4, _hip.DT_F16, _hip.DT_F32
    return _set(a, kw), _hip.lib().mdf_selective_step_dev, ()


def norm(**kw):
    a = ssm._Norm()
    a.s, a.out, a.post_weight, a.lds, a.ldo, a.rows, a.dim, a.groups, a.dtype, a.eps = P, 2 * P, 3 * P, 64, 64, 10, 64, 1, _hip.DT_F32, 1e-6
    a.scale = 1.0
    return _set(a, kw), _hip.lib().mdf_block_norm_dev, ()


def _set(a, kw):
    for k, v in kw.items():
        at = a
        *path, last = k.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, v)
    return a


@pytest.mark.parametrize("make, kw, what", [
    (conv, dict(dtype=_hip.DT_F64), "dtype"),
    (conv, dict(width=9), "width"),
    (conv, dict(width=0), "width"),
    (conv, dict(channels=0), "channels"),
    (conv, dict(x=None), "NULL"),
    (conv, dict(rows__lengths=None), "NULL"),
    (conv, dict(rows__B=-1), "sequences"),
    (conv, dict(rows__R=1 << 31), "rows"),
    (conv, dict(rows__max_len=101), "max_len"),
    (conv, dict(ldo=63), "stride"),
    (conv, dict(out=P + 64), "overlaps"),
    (conv, dict(out=P), "overlaps"),
    (conv, dict(state=3 * P, rows__n_slots=3), "states"),
    (scan, dict(dtype=_hip.DT_I32), "dtype"),
    (scan, dict(dt_dtype=_hip.DT_U8), "dtype"),
    (scan, dict(heads=5), "groups"),
    (scan, dict(groups=0), "groups"),
    (scan, dict(head_dim=257), "head_dim"),
    (scan, dict(state_dim=129), "state_dim"),
    (scan, dict(state_dim=0), "state_dim"),
    (scan, dict(c=None), "NULL"),
    (scan, dict(a=None), "NULL"),
    (scan, dict(ldy=127), "stride"),
    (scan, dict(ldb=-1), "stride"),
    (scan, dict(ldx=0), "stride"),
    (scan, dict(ldc=1 << 23), "stride"),
    (scan, dict(y=P + 2), "overlaps"),
    (scan, dict(y=2 * P), "overlaps"),
    (scan, dict(state=7 * P, rows__n_slots=2), "states"),
    (step, dict(width=9), "width"),
    (step, dict(n_slots=2), "states"),
    (step, dict(conv_state=None), "NULL"),
    (step, dict(y=P), "overlaps"),
    (step, dict(ldy=100), "stride"),
    (norm, dict(dim=0), "dim"),
    (norm, dict(dim=32769), "dim"),
    (norm, dict(groups=3), "groups"),
    (norm, dict(groups=2, pre_weight=4 * P), "pre-norm"),
    (norm, dict(gate_act=3), "gate_act"),
    (norm, dict(post_weight=None, post_bias=P), "post_bias"),
    (norm, dict(pre_bias=P), "pre_bias"),
    (norm, dict(scale_vec=P), "scale_vec"),
    (norm, dict(out=None), "NULL"),
    (norm, dict(residual=4 * P, residual_dtype=_hip.DT_F16, ldr=64, residual_out=5 * P, ldro=64), "type"),
    (norm, dict(residual=4 * P, residual_dtype=_hip.DT_F32, ldr=64), "NULL"),
    (norm, dict(out=P + 4), "overlaps"),
    (norm, dict(out=P, ldo=128), "overlaps"),
    (norm, dict(pre_weight=3 * P, residual=4 * P, residual_dtype=_hip.DT_F32, ldr=64, residual_out=2 * P, ldro=64), "outputs overlap"),
])
def test_c_entries_refuse(make, kw, what):
    a, fn, more = make(**kw)
    assert fn(ctypes.byref(a), *more, None) == _hip.MDF_EINVAL
    assert what in _hip.last_error()


def test_c_entries_refuse_null_and_accept_nothing_to_do():
    L = _hip.lib()
    for fn, more in ((L.mdf_causal_conv_dev, ()), (L.mdf_selective_scan_dev, (None, 0)), (L.mdf_selective_step_dev, ()), (L.mdf_block_norm_dev, ())):
        assert fn(None, *more, None) == _hip.MDF_EINVAL
    for make, kw in ((conv, dict(rows__B=0)), (conv, dict(rows__R=0, rows__max_len=0)), (scan, dict(rows__B=0)), (scan, dict(rows__R=0, rows__max_len=0)), (step, dict(B=0)), (norm, dict(rows=0))):
        a, fn, more = make(**kw)
        assert fn(ctypes.byref(a), *more, None) == _hip.MDF_OK, (make, kw)


def test_columns_of_one_wider_array_do_not_overlap():
    """y beside x in rows of one array (equal strides, disjoint columns): accepted, so the call gets as far as the device."""
    if _hip.device_count() > 0:
        pytest.skip("a GPU is visible")
    a, fn, more = conv(ldx=128, ldo=128, out=P + 64 * 4)
    assert fn(ctypes.byref(a), *more, None) == _hip.MDF_ENODEVICE
    a, fn, more = conv(ldx=128, ldo=128, out=P + 63 * 4)
    assert fn(ctypes.byref(a), *more, None) == _hip.MDF_EINVAL


def test_structures_have_the_headers_layout(tmp_path):
    """sizeof and the last member's offset of every argument structure, as the compiler lays include/mdfri.h out."""
    import os
    import shutil
    import subprocess
    from conftest import ROOT
    if not shutil.which("gcc"):
        pytest.skip("needs gcc")
    want = {"mdf_seq_rows": (ssm._Rows, "n_slots"), "mdf_conv_args": (ssm._Conv, "zero_skipped"), "mdf_scan_args": (ssm._Scan, "zero_skipped"), "mdf_step_args": (ssm._Step, "zero_skipped"),
            "mdf_block_norm_args": (ssm._Norm, "eps")}
    src = '#include <stdio.h>\n#include "mdfri.h"\nint main(void){%s return 0;}' % "".join(
        'printf("%%zu %%zu\\n", sizeof(%s), offsetof(%s, %s));' % (k, k, last) for k, (_, last) in want.items())
    (tmp_path / "t.c").write_text(src)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")])
    got = subprocess.check_output([str(tmp_path / "t")], text=True).split("\n")
    for line, (k, (cls, last)) in zip(got, want.items()):
        assert line == "%d %d" % (ctypes.sizeof(cls), getattr(cls, last).offset), k


def test_packed_heads_match_the_structures():
    """The addresses that every call packs end where the structures' strides begin."""
    assert ssm._CONV.size == ssm._Conv.ldx.offset and ssm._SCAN.size == ssm._Scan.ldx.offset and ssm._STEP.size == ssm._Step.ldx.offset and ssm._NORM.size == ssm._Norm.lds.offset
    a = ssm._Scan.from_buffer_copy(ssm._SCAN.pack(*range(1, 18)) + bytes(ctypes.sizeof(ssm._Scan) - ssm._SCAN.size))
    assert (a.rows.lengths, a.rows.positions, a.rows.R, a.rows.B, a.rows.max_len, a.rows.n_slots, a.x, a.dt, a.state, a.y) == (1, 4, 5, 6, 7, 8, 9, 12, 16, 17)


def test_python_layer_refuses_host_tensors_and_bad_rows():
    import torch
    rows = ssm.SequenceRows.build([3, 0, 5], device="cpu", align=16)
    assert rows.row_off.tolist() == [0, 16, 16, 32] and rows.max_len == 5 and not rows.dense
    assert ssm.SequenceRows.build([3, 0, 5], device="cpu").dense
    with pytest.raises(ValueError, match="not on a GPU"):
        ssm.causal_conv(torch.zeros(8, 4), torch.zeros(4, 4), rows)
    with pytest.raises(ValueError, match="not on a GPU"):
        ssm.block_norm(torch.zeros(8, 4))
    with pytest.raises(ValueError, match="float64"):
        ssm.causal_conv(torch.zeros(8, 4, dtype=torch.float64), torch.zeros(4, 4), rows)
    with pytest.raises(ValueError, match="none negative"):
        ssm.SequenceRows.build([3, -1], device="cpu")
    with pytest.raises(ValueError, match="int32"):
        ssm.SequenceRows(torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="one more"):
        ssm.SequenceRows(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="too many rows"):
        ssm.SequenceRows.build([2**30, 2**30], device="cpu")
    assert ssm.check_slots([2, -1, 0, -1], 3, device="cpu").tolist() == [2, -1, 0, -1]
    with pytest.raises(ValueError, match="share"):
        ssm.check_slots([1, 0, 1], 3, device="cpu")
    with pytest.raises(ValueError, match="outside"):
        ssm.check_slots([1, 3], 3, device="cpu")


def test_oracle_agrees_with_itself_token_by_token():
    """The 64-bit oracle: a prompt in one call == the same prompt in pieces through its kept states (what the kernels are held to as well)."""
    import ssm_oracle as o
    rng = np.random.default_rng(3)
    H, Pd, G, N, W, T = 4, 5, 2, 3, 3, 17
    C = H * Pd + 2 * G * N
    xbc, dt, a = rng.standard_normal((T, C)), rng.standard_normal((T, H)), -rng.uniform(0.5, 4, H)
    w, bias = rng.standard_normal((W, C)), rng.standard_normal(C)

    def block(rows, pos, ring, state):
        u, _ = o.conv(xbc[rows], w, bias, True, [len(rows)], [0], ring, None, [pos])
        return o.scan(u[:, :H * Pd].reshape(-1, H, Pd), dt[rows], a, u[:, H * Pd:H * Pd + G * N].reshape(-1, G, N), u[:, H * Pd + G * N:].reshape(-1, G, N), [len(rows)], [0], None, None,
                      state, None, [pos])[0]
    ring, state = np.zeros((1, W, C)), np.zeros((1, H, Pd, N))
    whole = block(np.arange(T), 0, ring.copy(), state.copy())
    parts, at = [], 0
    for n in (1, 1, 2, 5, 1, 7):
        parts.append(block(np.arange(at, at + n), at, ring, state))
        at += n
    assert np.allclose(np.concatenate(parts), whole, rtol=0, atol=1e-13)
