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
