"""Refusals of the paged-cache entry points: every one is answered before any
device work, so they run on CPU (the pointers are never followed)."""
import ctypes as C

import pytest
import torch

from heliopause_b200 import _lib, kernels as hk

P = 1 << 20  # an aligned address that is never followed


def _append(**kw):
    a = dict(k=P, ks=512, v=P, vs=512, q=P, qs=2048, in_dtype=0, rows=4, heads=8, kv_heads=2, dim=256, inv=P, half=128,
             qn=None, kn=None, norm_v=0, eps=1e-6, kc=P, vc=P, dtype=1, pages=10, page=16, table=P, width=4, starts=P,
             lens=P, seqs=2, out=P)
    a.update(kw)
    return _lib.lib().hpc_paged_kv_append(
        a["k"], a["ks"], a["v"], a["vs"], a["q"], a["qs"], a["in_dtype"], a["rows"], a["heads"], a["kv_heads"], a["dim"],
        a["inv"], a["half"], a["qn"], a["kn"], a["norm_v"], a["eps"], a["kc"], a["vc"], a["dtype"], a["pages"], a["page"],
        a["table"], a["width"], a["starts"], a["lens"], a["seqs"], a["out"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dim=80), hk.ERR_SHAPE), (dict(dim=0), hk.ERR_SHAPE), (dict(dim=512), hk.ERR_SHAPE),
    (dict(heads=3), hk.ERR_HEADS), (dict(kv_heads=0), hk.ERR_HEADS), (dict(heads=0), hk.ERR_HEADS),
    (dict(page=0), hk.ERR_SHAPE), (dict(page=24), hk.ERR_SHAPE), (dict(page=8), hk.ERR_SHAPE),
    (dict(page=2048), hk.ERR_SHAPE), (dict(pages=0), hk.ERR_SHAPE), (dict(pages=1 << 30), hk.ERR_SHAPE),
    (dict(width=0), hk.ERR_SHAPE), (dict(width=1 << 31), hk.ERR_SHAPE), (dict(rows=1 << 31), hk.ERR_SHAPE),
    (dict(seqs=1 << 21), hk.ERR_SHAPE), (dict(dtype=0), hk.ERR_TYPE), (dict(dtype=9), hk.ERR_TYPE),
    (dict(in_dtype=2), hk.ERR_TYPE), (dict(half=132), hk.ERR_SHAPE), (dict(half=129), hk.ERR_SHAPE),
    (dict(half=12), hk.ERR_SHAPE), (dict(ks=511), hk.ERR_SHAPE), (dict(vs=500), hk.ERR_SHAPE),
    (dict(ks=516), hk.ERR_SHAPE), (dict(qs=2040), hk.ERR_SHAPE), (dict(eps=-1.0), hk.ERR_ARG),
    (dict(eps=float("nan")), hk.ERR_ARG), (dict(k=None), hk.ERR_ARG), (dict(v=None), hk.ERR_ARG),
    (dict(kc=None), hk.ERR_ARG), (dict(table=None), hk.ERR_ARG), (dict(starts=None), hk.ERR_ARG),
    (dict(lens=None), hk.ERR_ARG), (dict(out=None), hk.ERR_ARG), (dict(inv=None), hk.ERR_ARG),
    (dict(k=P + 8), hk.ERR_ARG), (dict(kc=P + 2), hk.ERR_ARG), (dict(kn=P + 4), hk.ERR_ARG),
])
def test_append_refuses(kw, code):
    assert _append(**kw) == code
    assert _lib.last_error()


def test_append_of_nothing_needs_nothing():
    assert _append(rows=0, k=None, v=None, kc=None) == hk.OK
    assert _append(seqs=0, k=None, table=None) == hk.OK


def _paged(**kw):
    a = dict(q=P, qs=2048, kc=P, vc=P, dtype=1, pages=10, page=16, table=P, width=4, starts=P, lens=P, seqs=2, rows=4,
             heads=8, kv_heads=2, dim=256, mq=1, scale=1.0, window=0, ws=P, wsb=1 << 40, out=P, od=1, lse=None)
    a.update(kw)
    return _lib.lib().hpc_paged_attention(
        a["q"], a["qs"], a["kc"], a["vc"], a["dtype"], a["pages"], a["page"], a["table"], a["width"], a["starts"],
        a["lens"], a["seqs"], a["rows"], a["heads"], a["kv_heads"], a["dim"], a["mq"], a["scale"], a["window"], a["ws"],
        a["wsb"], a["out"], a["od"], a["lse"], None)


def _prompt(**kw):
    a = dict(q=P, qs=2048, k=P, ks=512, v=P, vs=512, dtype=1, starts=P, seqs=2, rows=4, heads=8, kv_heads=2, dim=256,
             mq=4, scale=1.0, window=0, ws=P, wsb=1 << 40, out=P, od=1, lse=None)
    a.update(kw)
    return _lib.lib().hpc_prompt_attention(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["dtype"], a["starts"], a["seqs"], a["rows"], a["heads"],
        a["kv_heads"], a["dim"], a["mq"], a["scale"], a["window"], a["ws"], a["wsb"], a["out"], a["od"], a["lse"], None)


BOTH = [
    (dict(dim=96), hk.ERR_SHAPE), (dict(heads=9), hk.ERR_HEADS), (dict(kv_heads=0), hk.ERR_HEADS),
    (dict(dtype=0), hk.ERR_TYPE), (dict(dtype=5), hk.ERR_TYPE), (dict(od=2), hk.ERR_TYPE), (dict(od=-1), hk.ERR_TYPE),
    (dict(qs=2044), hk.ERR_SHAPE), (dict(qs=2052), hk.ERR_SHAPE), (dict(rows=1 << 31), hk.ERR_SHAPE),
    (dict(window=1 << 31), hk.ERR_SHAPE), (dict(scale=float("nan")), hk.ERR_SHAPE), (dict(wsb=100), hk.ERR_SHAPE),
    (dict(q=None), hk.ERR_ARG), (dict(starts=None), hk.ERR_ARG), (dict(out=None), hk.ERR_ARG), (dict(ws=None), hk.ERR_ARG),
    (dict(q=P + 4), hk.ERR_ARG), (dict(out=P + 8), hk.ERR_ARG),
]


@pytest.mark.parametrize("kw,code", BOTH + [
    (dict(page=0), hk.ERR_SHAPE), (dict(page=48), hk.ERR_SHAPE), (dict(pages=0), hk.ERR_SHAPE), (dict(width=0), hk.ERR_SHAPE),
    (dict(table=None), hk.ERR_ARG), (dict(lens=None), hk.ERR_ARG), (dict(kc=None), hk.ERR_ARG), (dict(vc=P + 2), hk.ERR_ARG),
])
def test_paged_attention_refuses(kw, code):
    assert _paged(**kw) == code


@pytest.mark.parametrize("kw,code", BOTH + [
    (dict(ks=508), hk.ERR_SHAPE), (dict(vs=516), hk.ERR_SHAPE), (dict(k=None), hk.ERR_ARG), (dict(v=P + 8), hk.ERR_ARG),
])
def test_prompt_attention_refuses(kw, code):
    assert _prompt(**kw) == code


def test_workspace_query():
    n = C.c_size_t()
    L = _lib.lib()
    assert L.hpc_attention_workspace_bytes(8, 2, 256, C.byref(n)) == hk.OK and n.value > 0
    assert L.hpc_attention_workspace_bytes(8, 3, 256, C.byref(n)) == hk.ERR_HEADS
    assert L.hpc_attention_workspace_bytes(8, 2, 100, C.byref(n)) == hk.ERR_SHAPE
    assert L.hpc_attention_workspace_bytes(8, 2, 64, None) == hk.ERR_ARG
    assert _paged(rows=0, q=None, out=None) == hk.OK and _prompt(seqs=0, q=None, k=None) == hk.OK


def test_python_checks():
    f16 = dict(dtype=torch.float16)
    cache = torch.zeros((4, 16, 2, 64), **f16)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(hk.CudaKernelError):  # not on a device
        hk.paged_attention(torch.zeros((2, 4, 64), **f16), cache, cache, i32.view(1, 3), i32[:2], i32[:1], max_query_len=1,
                           scale=1.0)
    with pytest.raises(hk.CudaKernelError):
        hk.paged_kv_append(torch.zeros((2, 2, 64)), torch.zeros((2, 2, 64)), cache, cache[:2], i32.view(1, 3), i32[:2], i32[:1])
    with pytest.raises(hk.CudaKernelError):
        hk.prompt_attention(torch.zeros((2, 4, 64), **f16), torch.zeros((2, 2, 64), **f16), torch.zeros((2, 2, 64), **f16),
                            i32[:2], max_query_len=2, scale=1.0)
