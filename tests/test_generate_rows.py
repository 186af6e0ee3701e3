"""Rows that generate's sampling has no token for (the sampling kernel answers -1 for a NaN, or no logit above -inf): on the CPU."""
import torch

from kushkash_amd._generate import _admit, _by_kernel, _StopSignal


def test_a_row_without_a_token_is_counted_and_takes_a_valid_id():
    done, broken = torch.tensor([False, False, True, True]), torch.zeros(4, dtype=torch.bool)
    tok = _admit(torch.tensor([7, -1, -1, 3]), done, broken)
    assert tok.tolist() == [7, 0, 0, 3] and broken.tolist() == [False, True, False, False]
    assert _admit(torch.tensor([1, 2, 3, -1]), done, broken).tolist() == [1, 2, 3, 0]
    assert broken.tolist() == [False, True, False, False]                   # kept; a done row has nothing to draw


def test_rows_without_a_token_are_named():
    _StopSignal.check(torch.zeros(3, dtype=torch.bool))
    try:
        _StopSignal.check(torch.tensor([False, True, True]))
    except RuntimeError as e:
        assert "rows [1, 2]" in str(e) and "NaN" in str(e)
    else:
        raise AssertionError("no error")


def test_which_calls_draw_by_the_kernel():
    g = torch.Generator()
    assert not _by_kernel(False, 0.5, 0.1, g) and not _by_kernel(True, 1.0, 0.0, None) and not _by_kernel(True, 2.0, 0.0, None)
    assert _by_kernel(True, 0.9, 0.0, None) and _by_kernel(True, 1.0, 0.1, None) and _by_kernel(True, 1.0, 0.0, g)
