"""Values that are not finite in long caches: they reach the rows that see them
and no others, at no cost that grows with the keys."""
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
    hk.device_error()


def _check(b, q, window, scale, spots, out_dtype):
    """spots: (sequence, key, KV head, element, value).  Where rows see one, the
    result is it (or NaN for two that do not agree); everything else is as
    without them."""
    heads, dim = q.shape[1:]
    group = heads // b.key.shape[2]
    extra = torch.zeros((b.starts[-1], heads, dim), device="cuda")
    for s, j, h, d, x in spots:
        b.value.view(-1, b.key.shape[2], dim)[b.slots[s][j], h, d] = 1.0
    want, _, mag, smax = ref.attention(q, b.k_of, b.v_of, b.starts, b.lens, scale, window)
    for s, j, h, d, x in spots:
        v = b.value.view(-1, b.key.shape[2], dim)
        v[b.slots[s][j], h, d] = x
        a, e = b.starts[s], b.starts[s + 1]
        pos = torch.arange(b.lens[s] - (e - a), b.lens[s], device="cuda")
        sees = (pos >= j) & ((pos - j < window) if window else (pos >= j))
        extra[a:e][sees, h * group:(h + 1) * group, d] += x
    got = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(b.new), scale=scale,
                             window=window, out_dtype=out_dtype)
    hk.device_error()  # no wait gave up
    odd = ~torch.isfinite(extra)
    assert odd.any() and not odd.all()
    assert torch.equal(torch.nan_to_num(got[odd].float(), 7.0, 8.0, 9.0), torch.nan_to_num(extra[odd], 7.0, 8.0, 9.0))
    # (1.0 in their place changed the sums of rows that see them in that element only)
    tol = ref.attention_tolerance(q.dtype, out_dtype, mag, smax, dim, max(b.lens))
    assert ((got.double() - want).abs() <= tol)[~odd].all()


@pytest.mark.parametrize("dim,heads,kv_heads,dtype,window,out_dtype", [
    (256, 4, 2, torch.bfloat16, 0, torch.bfloat16),
    (256, 6, 2, torch.float16, 300, torch.float32),     # a group that does not divide a tile's rows
    (128, 4, 2, torch.float16, 0, torch.float16),
    (128, 4, 2, torch.bfloat16, 5000, torch.float32),
    (64, 8, 4, torch.bfloat16, 0, torch.bfloat16),
])
def test_long_keys_of_many_sequences(dim, heads, kv_heads, dtype, window, out_dtype):
    # too many items to cut their keys into parts
    new, lens = [130] * 40, [200] * 40
    lens[3], lens[17], lens[39] = 9000, 6001, 131
    b = ref.Batch(new, lens, kv_heads, dim, 64, dtype)
    q = _q(b, heads, dim, dtype)
    inf, nan = float("inf"), float("nan")
    spots = [(3, 8990, 0, 3, inf), (3, 8900, 1, 4, -inf), (3, 8950, 1, 4, inf), (17, 6000, 0, dim - 1, nan),
             (17, 5990, 1, 0, -inf), (39, 7, 0, 17, inf), (39, 130, 1, 17, nan)]
    _check(b, q, window, dim ** -0.5 / 4, spots, out_dtype)


@pytest.mark.parametrize("dim,dtype,out_dtype", [
    (64, torch.float16, torch.float32), (128, torch.bfloat16, torch.bfloat16), (256, torch.bfloat16, torch.bfloat16),
    (256, torch.float16, torch.float32)])
@pytest.mark.parametrize("window", [0, 2000])
def test_long_keys_in_parts(dim, dtype, out_dtype, window):
    b = ref.Batch([150], [12_000], 1, dim, 16, dtype)
    q = _q(b, 4, dim, dtype)
    inf, nan = float("inf"), float("nan")
    spots = [(0, 11_999, 0, 1, inf), (0, 11_900, 0, 8, -inf), (0, 11_875, 0, dim - 3, nan), (0, 11_860, 0, 40, inf)]
    if window:  # seen by the first rows only, and by a first part's rows
        spots += [(0, 12_000 - 150 - 2000 + 30, 0, 9, -inf), (0, 12_000 - 150 - 2000 + 1, 0, 10, nan)]
    _check(b, q, window, dim ** -0.5 / 4, spots, out_dtype)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_new_values_that_are_all_nan(dim):
    # an overflow upstream: every value of the last 40 tokens
    n, new, dtype = 5000, 200, torch.bfloat16
    b = ref.Batch([new, 140], [n, 140], 2, dim, 64, dtype)
    b.value.view(-1, 2, dim)[b.slots[0][n - 40:]] = torch.nan
    q = _q(b, 4, dim, dtype)
    got = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=new, scale=0.05)
    hk.device_error()
    assert torch.isnan(got[new - 40:new]).all() and torch.isfinite(got[:new - 40]).all() and torch.isfinite(got[new:]).all()
    b.value.nan_to_num_(0.0)
    want, _, mag, smax = ref.attention(q, b.k_of, b.v_of, b.starts, b.lens, 0.05, 0)
    tol = ref.attention_tolerance(dtype, dtype, mag, smax, dim, n)
    keep = torch.ones(b.rows, dtype=torch.bool, device="cuda")
    keep[new - 40:new] = False
    assert ((got.double() - want).abs() <= tol)[keep].all()


@pytest.mark.parametrize("dim,heads,kv_heads,window", [(64, 4, 1, 0), (128, 8, 2, 0), (128, 5, 1, 90), (256, 8, 2, 100)])
def test_packed_prompts_with_values_that_are_not_finite(dim, heads, kv_heads, window):
    new, dtype = [700, 1, 260], torch.float16
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn((sum(new), heads + 2 * kv_heads, dim), device="cuda", generator=g).to(dtype)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    starts = [0, 700, 701, 961]
    spots = [(0, 650, float("inf")), (0, 3, float("-inf")), (2, 100, float("nan")), (2, 259, float("inf"))]
    qs = torch.tensor(starts, dtype=torch.int32, device="cuda")
    extra = torch.zeros((961, heads, dim), device="cuda")
    for i, (s, j, val) in enumerate(spots):
        v[starts[s] + j, 0, 5 + i] = 1.0
    want, _, mag, smax = ref.attention(q, lambda s: k[starts[s]:starts[s + 1]], lambda s: v[starts[s]:starts[s + 1]], starts,
                                       new, 0.03, window)
    for i, (s, j, val) in enumerate(spots):
        v[starts[s] + j, 0, 5 + i] = val
        end = min(new[s], j + window) if window else new[s]
        extra[starts[s] + j:starts[s] + end, :heads // kv_heads, 5 + i] += val
    got = hk.prompt_attention(q, k, v, qs, max_query_len=700, scale=0.03, window=window)
    hk.device_error()
    odd = ~torch.isfinite(extra)
    assert torch.equal(torch.nan_to_num(got[odd].float(), 7.0, 8.0, 9.0), torch.nan_to_num(extra[odd], 7.0, 8.0, 9.0))
    assert ((got.double() - want).abs() <= ref.attention_tolerance(dtype, dtype, mag, smax, dim, 700))[~odd].all()
