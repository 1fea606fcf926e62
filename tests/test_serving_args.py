"""Refusals of the serving calls that are answered before any device work."""
import pytest

from heliopause_b200 import _lib, kernels as hk
from tests.test_paged_args import P, _append, _paged, _prompt


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_lengths_that_32_bits_do_not_hold_with_a_tile_behind_them(page):
    # a sequence's last tile ends up to 128 keys behind its last key
    most = (2 ** 31 - 1 - 1024) // page
    for call in (_append, _paged):
        assert call(page=page, width=most + 1) == hk.ERR_SHAPE and str(most + 1) in _lib.last_error()
        assert call(page=page, pages=most + 1) == hk.ERR_SHAPE
        # the largest is passed on, and refused for its missing pointer only
        assert call(page=page, width=most, pages=most, lens=None) == hk.ERR_ARG


# 4 rows of 8 heads of 256 in 16 bits are 16384 bytes, 2 KV heads 4096; the paged cache 10 pages of 16
Q, K, V, OUT = (P << i for i in range(1, 5))


@pytest.mark.parametrize("out,out_dtype", [
    (Q + 16, 1), (Q - 16, 1), (Q + 16384 - 16, 1), (Q - 16384 + 16, 1),
    (Q, 0), (Q - 32768 + 16, 0),  # f32 rows are twice as long
    (K, 1), (K - 16384 + 16, 1), (V, 1), (V + 4096 - 16, 1), (V - 32768 + 16, 0),
])
def test_outputs_over_inputs_are_refused(out, out_dtype):
    assert _paged(q=Q, kc=K, vc=V, out=out, od=out_dtype) == hk.ERR_ARG
    assert "lies over" in _lib.last_error()
    assert _prompt(q=Q, k=K, v=V, out=out, od=out_dtype) == hk.ERR_ARG
    assert "lies over" in _lib.last_error()


def test_outputs_over_the_end_of_a_cache_or_over_strided_queries_are_refused():
    cache = 10 * 16 * 2 * 256 * 2
    for kw in (dict(out=K + cache - 16), dict(out=V + cache - 16), dict(q=Q, out=Q, qs=2048 + 8)):
        assert _paged(**{**dict(q=Q, kc=K, vc=V), **kw}) == hk.ERR_ARG and "lies over" in _lib.last_error()
    for kw in (dict(out=K + 3 * 1024 * 2 + 1024 - 16), dict(out=V + 3 * 512 * 2 + 1024 - 16)):  # the last row's last bytes
        assert _prompt(**{**dict(q=Q, k=K, v=V, ks=1024), **kw}) == hk.ERR_ARG and "lies over" in _lib.last_error()
