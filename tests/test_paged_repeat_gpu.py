"""Attention gives the same bits every time, whichever block takes an item."""
import pytest
import torch

from heliopause_b200 import kernels as hk
from tests import paged_reference as ref
from tests.test_paged_gpu import _q

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    hk.init_device(0)


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 128, 4), (128, 28, 2), (256, 96, 3)])
@pytest.mark.parametrize("top", [300, 3000])
def test_same_bits_every_time(dim, heads, kv_heads, top):
    # more items than the machine holds, of many lengths: which block takes
    # which one, and behind how many tiles, is another matter every time
    g = torch.Generator().manual_seed(dim)
    new = [int(x) for x in torch.randint(1, 300, (16,), generator=g)]
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, top, (16,), generator=g))]
    b = ref.Batch(new, lens, kv_heads, dim, 64, torch.bfloat16)
    q = _q(b, heads, dim, torch.bfloat16, amp=6.0)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = None
    for i in range(40):
        if i % 4 == 0:
            flush.zero_()
        got = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(new),
                                 scale=dim ** -0.5, out_dtype=torch.float32, return_lse=True)
        first = first or got
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    hk.device_error()
