"""Refusals of the serving calls that are answered before any device work."""
import pytest

from heliopause_b200 import _lib, kernels as hk
from tests.test_paged_args import P, _append, _paged


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_lengths_that_32_bits_do_not_hold_with_a_tile_behind_them(page):
    # a sequence's last tile ends up to 128 keys behind its last key
    most = (2 ** 31 - 1 - 1024) // page
    for call in (_append, _paged):
        assert call(page=page, width=most + 1) == hk.ERR_SHAPE and str(most + 1) in _lib.last_error()
        assert call(page=page, pages=most + 1) == hk.ERR_SHAPE
        # the largest is passed on, and refused for its missing pointer only
        assert call(page=page, width=most, pages=most, lens=None) == hk.ERR_ARG
