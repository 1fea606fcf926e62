"""Refusals of hpc_logits_topk, answered before any device work."""
import ctypes as C

import pytest
import torch

from heliopause_b200 import _lib, kernels as hk

P = 1 << 20  # an address that is never followed


def _call(**kw):
    a = dict(x=P, stride=1000, rows=2, vocab=1000, k=8, h=P, hn=5, hs=P, pl=P, rep=P, fr=P, pr=P, bi=P, bv=P, bn=3, bs=P,
             al=P, als=32, ws=P, wsb=1 << 30, ids=P, vals=P)
    a.update(kw)
    return _lib.lib().hpc_logits_topk(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=0), hk.ERR_SHAPE), (dict(k=65), hk.ERR_SHAPE), (dict(vocab=5, k=6), hk.ERR_SHAPE), (dict(vocab=0), hk.ERR_SHAPE),
    (dict(vocab=(1 << 20) + 1), hk.ERR_SHAPE), (dict(rows=65536), hk.ERR_SHAPE), (dict(stride=999), hk.ERR_SHAPE),
    (dict(als=31), hk.ERR_SHAPE), (dict(wsb=127), hk.ERR_SHAPE), (dict(x=None), hk.ERR_ARG), (dict(ws=None), hk.ERR_ARG),
    (dict(ids=None), hk.ERR_ARG), (dict(vals=None), hk.ERR_ARG), (dict(hs=None), hk.ERR_ARG), (dict(bv=None), hk.ERR_ARG),
    (dict(bs=None), hk.ERR_ARG), (dict(ws=P + 4), hk.ERR_ARG),
])
def test_refuses(kw, code):
    assert _call(**kw) == code
    assert _lib.last_error()


def test_no_rows_and_workspace_query():
    assert _call(rows=0, x=None, ids=None, wsb=0) == hk.OK
    n = C.c_size_t()
    assert _lib.lib().hpc_logits_topk_workspace_bytes(3, 5000, 7, C.byref(n)) == hk.OK and n.value >= 3 * 7 * 8
    assert _lib.lib().hpc_logits_topk_workspace_bytes(3, 5000, 7, None) == hk.ERR_ARG


def test_python_checks():
    x = torch.zeros((2, 100))
    with pytest.raises(hk.CudaKernelError):  # not on a device
        hk.logits_topk(x, 4)
    with pytest.raises(hk.CudaKernelError):
        hk.logits_topk(x.half(), 4)
