"""Arguments at the ends of their ranges."""
import pytest
import torch

from heliopause_b200 import kernels as hk
from tests import paged_reference as ref
from tests.test_paged_gpu import _check, _q

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    hk.init_device(0)
    yield
    hk.device_error()


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 2), (128, 4, 2), (256, 2, 1)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 31 - 40, 6])
@pytest.mark.parametrize("new,lens", [([8, 1, 10], [5, 1, 0]), ([60, 8, 300], [50, 5, 263]), ([150], [3])])
def test_wide_windows_and_rows_before_the_first_key(dim, heads, kv_heads, window, new, lens):
    # rows at negative positions see nothing, the others every key up to their own
    b = ref.Batch(new, lens, kv_heads, dim, 16, torch.bfloat16)
    q = _q(b, heads, dim, torch.bfloat16)
    for hint in (1, max(new)):
        got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=hint,
                                      scale=dim ** -0.5, window=window, return_lse=True)
        _check(got, lse, b, q, dim ** -0.5, window)
