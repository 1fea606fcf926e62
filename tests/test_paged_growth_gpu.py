"""Rows whose largest score comes late: the running maximum grows by more than the
kernel lets pass and what was summed so far is rescaled, while the values of the
tiles before may still be on their way."""
import pytest
import torch

from heliopause_b200 import kernels as hk
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    hk.init_device(0)
    yield
    hk.device_error()


def _aim(q, k_of, starts, lens, scale, seed):
    """Every second row of q points at keys of its own: one, or one after the other with
    ever larger scores (9, 18, 27 ... in log2 units, above the rest)."""
    rows, heads, dim = q.shape
    g = torch.Generator().manual_seed(seed)
    for s, n in enumerate(lens):
        k = k_of(s).float()
        group = heads // k.shape[1]
        for r in range(starts[s], starts[s + 1], 2):
            pos = n - (starts[s + 1] - r)
            for h in range(heads):
                at = torch.randint(0, pos + 1, (1 + (r // 2 + h) % 4,), generator=g).sort().values.tolist()
                x = sum(k[j, h // group] / k[j, h // group].square().sum() * (9.5 * (i + 1) * 0.6931 / scale)
                        for i, j in enumerate(at))
                q[r, h] = (q[r, h].float() * 0.2 + x).to(q.dtype)


def _tolerance(q, v_of, starts, lens, mag, smax):
    """attention_tolerance, and what it leaves out: f16 probabilities below 2^-14 are
    rounded by half of 2^-24, whatever their size.  They are relative to a maximum
    that is never above the row's, so their sum is 1 at least, and an element is off
    by 2^-25 of the sum of its |v| at most.  (bf16 has f32's exponents.)"""
    tol = ref.attention_tolerance(q.dtype, q.dtype, mag, smax, q.shape[-1], max(lens))
    if q.dtype is torch.float16:
        for s in range(len(lens)):
            v = v_of(s).double().abs().sum(0)
            tol[starts[s]:starts[s + 1]] += 2.0 ** -25 * v.repeat_interleave(q.shape[1] // v.shape[0], 0)
    return tol


@pytest.mark.parametrize("dim,heads,kv_heads,dtype,page,new,lens", [
    (128, 10, 2, torch.float16, 16, [202, 1], [1739, 1417]),
    (128, 16, 4, torch.bfloat16, 64, [100, 5, 121, 40], [1999, 2338, 1142, 1048]),
    (128, 4, 2, torch.bfloat16, 16, [150], [1100]),
    (64, 8, 2, torch.float16, 16, [160, 33], [1500, 2000]),
    (64, 4, 4, torch.bfloat16, 64, [130], [700]),
    (256, 8, 2, torch.bfloat16, 16, [160, 1], [1700, 900]),
    (256, 4, 2, torch.float16, 64, [128], [900]),
])
def test_maxima_that_grow_late(dim, heads, kv_heads, dtype, page, new, lens):
    scale = dim ** -0.5
    b = ref.Batch(new, lens, kv_heads, dim, page, dtype)
    q = torch.randn((b.rows, heads, dim), device="cuda", generator=b.gen).to(dtype)
    _aim(q, b.k_of, b.starts, b.lens, scale, dim)
    want, _, mag, smax = ref.attention(q, b.k_of, b.v_of, b.starts, b.lens, scale, 0)
    tol = _tolerance(q, b.v_of, b.starts, b.lens, mag, smax)
    other = ref.Batch([1] * 8, [3000] * 8, 2, 128, 64, torch.float16, seed=9)
    oq = torch.randn((8, 8, 128), device="cuda", generator=other.gen).half()
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    outs = []
    for i in range(60):
        if i % 3 == 0:
            flush.zero_()  # keys and values from memory
        if i % 2:  # another kernel before, whose blocks leave one after the other
            hk.paged_attention(oq, other.key, other.value, other.table, other.query_starts, other.kv_lens, max_query_len=1,
                               scale=0.1)
        outs.append(hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(new),
                                       scale=scale))
    for o in outs:
        assert ((o.double() - want).abs() <= tol).all()
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("dim,heads,kv_heads,dtype,new", [
    (64, 4, 1, torch.bfloat16, [300, 700]), (128, 8, 2, torch.float16, [600, 130]), (256, 2, 1, torch.bfloat16, [900])])
def test_maxima_that_grow_late_in_packed_prompts(dim, heads, kv_heads, dtype, new):
    scale = dim ** -0.5
    b = ref.Batch(new, new, kv_heads, dim, 16, dtype)
    k, v = (torch.cat([f(s) for s in range(len(new))]) for f in (b.k_of, b.v_of))
    q = torch.randn((b.rows, heads, dim), device="cuda", generator=b.gen).to(dtype)
    _aim(q, b.k_of, b.starts, b.lens, scale, dim)
    want, _, mag, smax = ref.attention(q, b.k_of, b.v_of, b.starts, b.lens, scale, 0)
    tol = _tolerance(q, b.v_of, b.starts, b.lens, mag, smax)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    outs = []
    for i in range(30):
        if i % 3 == 0:
            flush.zero_()
        outs.append(hk.prompt_attention(q, k, v, b.query_starts, max_query_len=max(new), scale=scale))
    for o in outs:
        assert ((o.double() - want).abs() <= tol).all()
        assert torch.equal(o, outs[0])
