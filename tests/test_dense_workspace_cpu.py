"""What mla_prefill asks for as workspace: room for the pieces that a call can have, no more."""
import pytest

ROW = 128 * 4 + 8                                      # a row of a piece: 128 values, maximum and sum


def _pieces(lib, *sizes):
    n = lib.litedsa_mla_prefill_workspace(*sizes)
    assert n == 0 or (n - 16) % (256 * ROW) == 0
    return max(n - 16, 0) // (256 * ROW)


@pytest.mark.parametrize("Tq,Tk,heads,most", [
    (1, 385, 1, 2),                                    # one tile of four blocks: two pieces of two
    (1, 385, 4, 8), (3, 1000, 1, 12), (3, 1281, 2, 30), (1, 512, 16, 32),
])
def test_short_calls(built_lib, Tq, Tk, heads, most):
    assert 2 <= _pieces(built_lib, Tq, Tk, heads) <= most


def test_other_calls(built_lib):
    full = _pieces(built_lib, 4096, 32768, 16)         # four a multiprocessor
    assert full >= 4 and full % 4 == 0
    assert _pieces(built_lib, 300, 9001, 8) == _pieces(built_lib, 64, 4096, 16) == full
    assert _pieces(built_lib, 1, 1 << 20, 1) == full   # a tile in as many pieces as there is room for
    assert _pieces(built_lib, 1, 384, 1) == _pieces(built_lib, 4096, 384, 16) == _pieces(built_lib, 1 << 20, 4096, 16) == 0
