"""The state-space block's operators without a GPU: calls at the edges of what their documentation allows."""
import pytest

from mDeepFRI import ssm


class _Maker:
    """Stands for an input: says how an output like it would be made."""

    def new_empty(self, shape):
        return "empty"

    def new_zeros(self, shape):
        return "zeros"


@pytest.mark.parametrize("lengths, align, total, want", [([3, 0, 5], 1, 8, "empty"), ([3, 0, 5], 1, 9, "zeros"), ([3, 5], 16, 32, "zeros"), ([], 1, 4, "zeros"), ([0, 0], 1, 1, "zeros"), ([16, 32], 16, 48, "empty"),
                                                         ([16, 32], 16, 64, "zeros")])
def test_an_output_with_rows_of_no_sequence_is_made_of_zeros(lengths, align, total, want):
    """Rows behind the last sequence count too: an array may be longer than the sequences in it (a buffer of one size for every batch)."""
    rows = ssm.SequenceRows.build(lengths, device="cpu", align=align)
    assert ssm._made(None, _Maker(), rows, (total, 7)) == want
    assert ssm._made("given", _Maker(), rows, (total, 7)) == "given"


def test_the_callers_word_on_dense_rows():
    built = ssm.SequenceRows.build([2, 3], device="cpu")
    for total, made in ((None, "empty"), (5, "empty"), (4, "zeros")):
        assert ssm._made(None, _Maker(), ssm.SequenceRows(built.lengths, built.row_off, 3, dense=True, total=total), (5, 7)) == made
    assert ssm._made(None, _Maker(), ssm.SequenceRows(built.lengths, built.row_off, 3), (5, 7)) == "zeros"


def _norm_calls(monkeypatch):
    """block_norm's argument structures as the library would get them, from tensors on the host."""
    seen = []
    monkeypatch.setattr(ssm, "_call", lambda fn, device, args: seen.append(ssm._Norm.from_buffer_copy(args)))
    monkeypatch.setattr(ssm, "_matrix", lambda t, *a: t.stride(0))
    return seen


@pytest.mark.parametrize("kind", ["array", "tensor"])
def test_a_scale_or_eps_changed_in_place_is_read_again(monkeypatch, kind):
    import numpy as np
    import torch
    seen = _norm_calls(monkeypatch)
    s, r, w = torch.zeros(3, 8), torch.zeros(3, 8), torch.ones(8)
    make = (lambda v: np.array(v)) if kind == "array" else (lambda v: torch.tensor(v, dtype=torch.float64))
    scale, eps, groups = make(0.5), make(1e-5), np.array(2)
    for k, e, g in ((0.5, 1e-5, 2), (0.25, 1e-5, 2), (0.25, 0.125, 2), (0.25, 0.125, 4), (-2.0, 1e-6, 1)):
        scale[...], eps[...], groups[...] = k, e, g
        ssm.block_norm(s, residual=r, post_weight=w, scale=scale, eps=eps, groups=groups)
        got = seen.pop()
        assert (got.scale, got.groups, got.dim, got.rows) == (k, g, 8, 3) and got.eps == np.float32(e)


def test_signs_and_odd_numbers_of_scale(monkeypatch):
    import math
    import torch
    seen = _norm_calls(monkeypatch)
    for k in (0.0, -0.0, 1, True, math.inf, math.nan, 1e39):
        ssm.block_norm(torch.zeros(3, 8), residual=torch.zeros(3, 8), scale=k)
        got, k = seen.pop().scale, math.inf if k == 1e39 else k       # (beyond float32)
        assert math.copysign(1, got) == math.copysign(1, k) and (got == k or (got != got and k != k))


def test_a_scale_on_a_gpu_is_refused():
    """Reading it would wait for the GPU."""
    import torch

    class OnGpu:
        is_cuda, device = True, "cuda:0"
    with pytest.raises(ValueError, match="scale.*host"):
        ssm.block_norm(torch.zeros(3, 8), scale=OnGpu())
    with pytest.raises(ValueError, match="eps.*host"):
        ssm.block_norm(torch.zeros(3, 8), eps=OnGpu())
    with pytest.raises(ValueError, match="groups.*host"):
        ssm.block_norm(torch.zeros(3, 8), groups=OnGpu())


def _scan_args(R, B, max_len, heads=16, groups=1, head_dim=64, state_dim=128):
    from mDeepFRI import _hip
    P, a = 1 << 40, ssm._Scan()                        # addresses that nothing reads
    a.rows.lengths, a.rows.row_off, a.rows.R, a.rows.B, a.rows.max_len = P, P, R, B, max_len
    a.x, a.b, a.c, a.dt, a.a, a.y = (k * P for k in range(1, 7))
    a.ldx = a.ldy = heads * head_dim
    a.ldb = a.ldc = groups * state_dim
    a.lddt, a.heads, a.groups, a.head_dim, a.state_dim, a.dtype, a.dt_dtype = heads, heads, groups, head_dim, state_dim, _hip.DT_BF16, _hip.DT_BF16
    return a


@pytest.mark.parametrize("short", [0, 1, 32, 128, 5000, 70000])
def test_a_long_prompt_beside_many_short_sequences_is_cut_all_the_same(short):
    """The workspace goes by the rows, not by sequences times segments, and no number of sequences refuses the cut."""
    import ctypes
    from mDeepFRI import _hip
    a = _scan_args(32768 + short, 1 + short, 32768)
    need = _hip.lib().mdf_scan_workspace_bytes(ctypes.byref(a))
    state = 16 * 64 * 128 * 4
    assert 32 * state < need <= 65 << 20
    if _hip.device_count() == 0:
        assert _hip.lib().mdf_selective_scan_dev(ctypes.byref(a), 1 << 45, need, None) == _hip.MDF_ENODEVICE
    assert _hip.lib().mdf_selective_scan_dev(ctypes.byref(a), 1 << 45, need - 1, None) == _hip.MDF_ECAPACITY


def test_workspace_of_the_scan_is_bounded():
    """Any sizes: at most 65 MiB, none where no sequence is long."""
    import ctypes
    import random
    from mDeepFRI import _hip
    rng = random.Random(7)
    for _ in range(2000):
        groups = rng.choice([1, 1, 2, 8])
        R, heads = rng.choice([600, 5000, 40000, 10**6, 2**31 - 1]), groups * rng.choice([1, 2, 16, 128, 4096])
        a = _scan_args(R, rng.choice([1, 7, 1000]), rng.choice([0, 512, 513, R // 3, R]), heads, groups, rng.choice([1, 32, 40, 64, 256]), rng.choice([1, 16, 128]))
        if a.heads * a.head_dim >= 1 << 23:
            continue
        need = _hip.lib().mdf_scan_workspace_bytes(ctypes.byref(a))
        assert need <= 65 << 20 and (need == 0 or a.rows.max_len > 512), (R, heads, a.rows.max_len)


@pytest.mark.parametrize("channels, fits", [(8 * 127, True), (8 * 127 + 1, False)])
def test_a_convolution_larger_than_a_grid_is_refused(channels, fits):
    """A dimension of a grid holds fewer than 2^32 threads: 2^28 rows are 2^25 tiles, of 128 lanes for 1 017 and more bfloat16 channels."""
    from mDeepFRI import _hip
    a = ssm._Conv()
    a.rows.lengths, a.rows.row_off, a.rows.R, a.rows.B, a.rows.max_len = 1 << 40, 1 << 40, 1 << 28, 1, 1 << 28
    a.x, a.weight, a.out, a.ldx, a.ldo, a.channels, a.width, a.dtype = 1 << 41, 1 << 40, 1 << 45, channels, channels, channels, 2, _hip.DT_BF16
    if fits and _hip.device_count() > 0:
        pytest.skip("a GPU is visible")
    import ctypes
    rc = _hip.lib().mdf_causal_conv_dev(ctypes.byref(a), None)
    assert rc == (_hip.MDF_ENODEVICE if fits else _hip.MDF_EINVAL) and (fits or "too many" in _hip.last_error())


@pytest.mark.parametrize("sequences, fits", [(2**23 - 1, True), (2**28 - 8, True), (2**28, False)])
def test_a_scan_of_more_workgroups_than_the_library_counts_is_refused(sequences, fits):
    """2^31 workgroups: 8 per sequence here; every smaller number takes as many rows of the grid as it needs."""
    import ctypes
    from mDeepFRI import _hip
    a = _scan_args(2**31 - 1, sequences, 1)
    if fits and _hip.device_count() > 0:
        pytest.skip("a GPU is visible")
    rc = _hip.lib().mdf_selective_scan_dev(ctypes.byref(a), None, 0, None)
    assert rc == (_hip.MDF_ENODEVICE if fits else _hip.MDF_EINVAL) and (fits or "too many" in _hip.last_error())


def _calls():
    """Every operator with small arguments of the right forms: name -> (function, positional, keyword)."""
    import torch
    rows = ssm.SequenceRows.build([3, 2], device="cpu")
    z, h = torch.zeros, dict(d=torch.zeros(2), dt_bias=torch.zeros(2))
    return {
        "causal_conv": (ssm.causal_conv, dict(x=z(5, 8), weight=z(4, 8), rows=rows), dict(bias=z(8), state=z(2, 4, 8), out=z(5, 8))),
        "selective_scan": (ssm.selective_scan, dict(x=z(5, 2, 4), dt=z(5, 2), a=z(2), b=z(5, 1, 3), c=z(5, 1, 3), rows=rows), dict(h, state=z(2, 2, 4, 3), out=z(5, 2, 4))),
        "selective_step": (ssm.selective_step, dict(xbc=z(2, 14), dt=z(2, 2), a=z(2)), dict(h, conv_weight=z(4, 14), conv_bias=z(14), conv_state=z(2, 4, 14), state=z(2, 2, 4, 3), out=z(2, 2, 4))),
        "block_norm": (ssm.block_norm, dict(s=z(5, 8)), dict(residual=z(5, 8), gate=z(5, 8), post_weight=z(8), post_bias=z(8), scale_vec=z(8), pre_weight=z(8), pre_bias=z(8), residual_out=z(5, 8),
                                                           out=z(5, 8))),
    }


@pytest.mark.parametrize("op", ["causal_conv", "selective_scan", "selective_step", "block_norm"])
def test_every_tensor_with_a_tangent_is_refused(op):
    """A forward-mode derivative would be lost without a word; also under no_grad, which does not stop forward mode."""
    import torch
    from torch.autograd import forward_ad
    fn, args, more = _calls()[op]
    args = {**args, **more}
    with forward_ad.dual_level():
        for name, t in args.items():
            if not torch.is_tensor(t):
                continue
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(ValueError, match=name + " carries a tangent"):
                fn(**{**args, name: dual})
            with torch.no_grad(), pytest.raises(ValueError, match=name + " carries a tangent"):
                fn(**{**args, name: dual})
        with pytest.raises(ValueError, match="not on a GPU"):        # none of them: the next check
            fn(**args)


def test_checked_tensors_of_rows_cannot_be_exchanged():
    """The kernels go by the number of sequences that was checked: shorter tensors put in its place would be read past their ends."""
    import torch
    rows = ssm.SequenceRows.build([3, 0, 5], device="cpu")
    for name in ("lengths", "row_off", "count", "form"):
        with pytest.raises(AttributeError):
            setattr(rows, name, torch.zeros(1, dtype=torch.int32))
    assert rows.lengths.tolist() == [3, 0, 5] and rows.row_off.tolist() == [0, 3, 3, 8] and rows.count == 3 and rows.form == (3, -1)
    rows.max_len = 7                                  # another batch of three in the same tensors
    assert rows.max_len == 7


@pytest.mark.parametrize("op", ["causal_conv", "selective_scan", "selective_step"])
def test_a_pool_without_slots_is_refused(op, monkeypatch):
    """An empty tensor has no address, which to the library is a call without states: it would run what has to be skipped."""
    import torch
    monkeypatch.setattr(ssm, "_matrix", lambda t, *a: t.stride(0))
    monkeypatch.setattr(ssm, "_call", lambda fn, device, *args: None)
    fn, args, more = _calls()[op]
    args = {**args, **more}
    fn(**args)
    for name in ("state", "conv_state"):
        if name in args:
            with pytest.raises(ValueError, match="no slot"):
                fn(**{**args, name: args[name][:0], "slots": torch.full((2,), -1, dtype=torch.int32)})
    if op != "selective_step":
        nobody = dict(args, rows=ssm.SequenceRows.build([], device="cpu"), state=args["state"][:0])
        assert torch.equal(fn(**nobody), args["out"])
