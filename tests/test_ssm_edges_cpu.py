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
