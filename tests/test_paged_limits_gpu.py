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


@pytest.mark.parametrize("dim,heads,kv_heads,new,lens", [
    (64, 4, 2, [1] * 9, [1, 70, 400, 3, 900, 0, 64, 65, 2000]),    # few rows, some keys in parts
    (128, 8, 2, [5] * 4, [5, 700, 66, 3000]),
    (256, 6, 2, [130, 1, 300], [130, 40, 900]),                    # many rows
    (128, 4, 1, [100], [6000]),                                    # and their keys in parts
])
def test_output_in_the_place_of_the_queries(dim, heads, kv_heads, new, lens):
    b = ref.Batch(new, lens, kv_heads, dim, 16, torch.bfloat16)
    if b.lens[0] > 100:  # a value that some rows see and that is not finite
        b.value.view(-1, kv_heads, dim)[b.slots[0][-20], 0, 3] = torch.inf
    q = _q(b, heads, dim, torch.bfloat16)

    def call(x, out):
        return hk.paged_attention(x, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(new),
                                  scale=dim ** -0.5, out=out)

    want = call(q, None)
    for _ in range(10):
        x = q.clone()
        assert call(x, x) is x and torch.equal(x, want)
    n = torch.tensor(new).sum().item()
    k, v = (torch.randn((n, kv_heads, dim), device="cuda", generator=b.gen).bfloat16() for _ in range(2))
    want = hk.prompt_attention(q, k, v, b.query_starts, max_query_len=max(new), scale=0.05)
    x = q.clone()
    hk.prompt_attention(x, k, v, b.query_starts, max_query_len=max(new), scale=0.05, out=x)
    assert torch.equal(x, want)
    for over in (k, v):
        with pytest.raises(hk.CudaKernelError):
            hk.prompt_attention(q[:, :kv_heads].contiguous(), k, v, b.query_starts, max_query_len=max(new), scale=0.05, out=over)
