"""Paged KV cache on the GPU: append (norms, rotation, write), attention of
the newest rows over the pages, attention over packed prompts -- against plain
64-bit forms."""
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
    hk.device_error()  # no batch here points outside its buffers


def _q(b, heads, dim, dtype, strided=False, amp=1.5):
    q = torch.randn((b.rows, heads + (3 if strided else 0), dim), device="cuda", generator=b.gen) * amp
    return q.to(dtype)[:, :heads]


def _check(got, lse, b, q, scale, window, out_dtype=None):
    want, want_lse, mag, smax = ref.attention(q, b.k_of, b.v_of, b.starts, b.lens, scale, window)
    n = b.starts[-1]
    tol = ref.attention_tolerance(q.dtype, out_dtype or q.dtype, mag, smax, q.shape[-1], max([1] + b.lens))
    d = (got.double() - want).abs()[:n]
    assert torch.isfinite(got[:n]).all()
    assert (d <= tol[:n]).all(), f"off by {(d / tol[:n].clamp_min(1e-30)).max().item():.3g} of the tolerance"
    if lse is not None:
        fin = torch.isfinite(want_lse[:n])
        assert torch.equal(torch.isfinite(lse[:n]), fin)
        dl = (lse[:n].double() - want_lse[:n])[fin].abs()
        lt = (q.shape[-1] * 2.0 ** -23 * smax[:n] + 2.0 ** -18 + 2.0 ** -21 * want_lse[:n].abs())[fin]
        assert (dl <= lt).all()


LENS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 130, 300, 1025]


@pytest.mark.parametrize("dim,dtype,heads,kv_heads,page,window", [
    (64, torch.float16, 8, 8, 16, 0),
    (64, torch.bfloat16, 14, 2, 64, 33),
    (128, torch.float16, 32, 8, 16, 0),
    (128, torch.bfloat16, 16, 1, 128, 0),
    (128, torch.bfloat16, 24, 1, 32, 1),
    (256, torch.float16, 8, 2, 16, 0),
    (256, torch.bfloat16, 8, 2, 64, 100),
    (256, torch.bfloat16, 16, 2, 1024, 0),
])
def test_decode_over_pages(dim, dtype, heads, kv_heads, page, window):
    b = ref.Batch([1] * len(LENS), LENS, kv_heads, dim, page, dtype, spare_rows=3)
    q = _q(b, heads, dim, dtype, strided=True)
    out = torch.full((b.rows, heads, dim), 7.0, dtype=dtype, device="cuda")
    got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=1,
                                  scale=dim ** -0.5, window=window, out=out, return_lse=True)
    assert got is out and (out[b.starts[-1]:] == 7.0).all()  # rows of no sequence are left
    _check(got, lse, b, q, dim ** -0.5, window)


@pytest.mark.parametrize("dim,dtype,heads,kv_heads,page,window", [
    (64, torch.bfloat16, 4, 4, 16, 0),
    (128, torch.float16, 32, 8, 64, 9),
    (256, torch.float16, 8, 2, 16, 0),
    (256, torch.bfloat16, 8, 1, 32, 3),
])
def test_several_new_rows_empty_rows_and_sequences(dim, dtype, heads, kv_heads, page, window):
    # no key at all, fewer keys than new rows (leading rows see nothing), no new rows
    new = [5, 1, 3, 0, 8, 2, 5, 0, 7]
    lens = [5, 0, 2, 40, 200, 66, 1000, 0, 71]
    b = ref.Batch(new, lens, kv_heads, dim, page, dtype)
    q = _q(b, heads, dim, dtype)
    got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=8,
                                  scale=0.07, window=window, out_dtype=torch.float32, return_lse=True)
    _check(got, lse, b, q, 0.07, window, torch.float32)
    assert (got[5] == 0).all() and (lse[5] == -torch.inf).all() and (got[6] == 0).all()


@pytest.mark.parametrize("dim,dtype,heads,kv_heads,page,new,lens,window", [
    (64, torch.float16, 4, 2, 16, [200, 33, 129], [200, 500, 130], 0),
    (64, torch.bfloat16, 6, 2, 32, [64, 128], [700, 128], 70),
    (128, torch.bfloat16, 8, 2, 16, [300, 1, 17], [300, 900, 18], 0),
    (128, torch.float16, 8, 8, 128, [129, 140], [260, 1000], 128),
    (256, torch.bfloat16, 8, 2, 64, [130, 257, 9], [131, 800, 300], 0),
    (256, torch.float16, 4, 1, 16, [255], [256], 40),
    (256, torch.float16, 4, 4, 256, [100, 0, 150], [90, 0, 350], 0),
])
def test_chunks_over_pages(dim, dtype, heads, kv_heads, page, new, lens, window):
    b = ref.Batch(new, lens, kv_heads, dim, page, dtype, spare_rows=2)
    q = _q(b, heads, dim, dtype, strided=True)
    out = torch.full((b.rows, heads, dim), 7.0, dtype=dtype, device="cuda")
    got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(new),
                                  scale=dim ** -0.5, window=window, out=out, return_lse=True)
    assert (out[b.starts[-1]:] == 7.0).all()
    _check(got, lse, b, q, dim ** -0.5, window)


class _Packed:
    def __init__(self, new, kv_heads, dim, dtype, heads, spare=0, seed=0):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens = list(new)
        self.starts = [sum(new[:i]) for i in range(len(new) + 1)]
        self.rows = self.starts[-1] + spare
        x = torch.randn((self.rows, heads + 2 * kv_heads, dim), device="cuda", generator=self.gen).to(dtype)
        x[self.starts[-1]:] = torch.nan  # rows behind the last sequence
        self.q, self.k, self.v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
        self.query_starts = torch.tensor(self.starts, dtype=torch.int32, device="cuda")

    def k_of(self, s):
        return self.k[self.starts[s]:self.starts[s + 1]]

    def v_of(self, s):
        return self.v[self.starts[s]:self.starts[s + 1]]


@pytest.mark.parametrize("dim,dtype,heads,kv_heads,new,window", [
    (64, torch.float16, 4, 4, [1], 0),
    (64, torch.bfloat16, 7, 1, [130, 1, 64, 0, 257], 0),
    (128, torch.float16, 8, 2, [128, 300, 2, 127], 0),
    (128, torch.bfloat16, 4, 2, [1000, 129], 200),
    (128, torch.bfloat16, 4, 2, [5, 3, 1], 0),
    (256, torch.float16, 8, 2, [333], 0),
    (256, torch.bfloat16, 8, 2, [700, 1, 128, 129], 0),
    (256, torch.bfloat16, 2, 1, [513, 256], 64),
    (256, torch.float16, 2, 2, [400], 1),
])
def test_packed_prompts(dim, dtype, heads, kv_heads, new, window):
    b = _Packed(new, kv_heads, dim, dtype, heads, spare=5)
    out = torch.full((b.rows, heads, dim), 7.0, dtype=dtype, device="cuda")
    got, lse = hk.prompt_attention(b.q, b.k, b.v, b.query_starts, max_query_len=max(new), scale=dim ** -0.5,
                                   window=window, out=out, return_lse=True)
    assert (out[b.starts[-1]:] == 7.0).all()
    _check(got, lse, b, b.q, dim ** -0.5, window)


@pytest.mark.parametrize("dim,heads,kv_heads,window", [(64, 16, 8, 0), (128, 8, 8, 50), (256, 12, 6, 0)])
def test_more_tiles_than_the_machine_holds_at_once(dim, heads, kv_heads, window):
    # several times the tiles of one wave, of all lengths, among them sequences
    # without keys, and rows before the first key
    g = torch.Generator().manual_seed(dim)
    new = torch.randint(0, 500, (60,), generator=g).tolist()
    past = [(-20, 0, 0, 130, 411)[i % 5] if n else 0 for i, n in enumerate(new)]
    lens = [max(0, n + p) for n, p in zip(new, past)]
    b = ref.Batch(new, lens, kv_heads, dim, 16, torch.bfloat16)
    q = _q(b, heads, dim, torch.bfloat16)
    for rep in range(3):
        got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=500,
                                      scale=-(dim ** -0.5), window=window, return_lse=True)
        if rep == 0:
            _check(got, lse, b, q, -(dim ** -0.5), window)
            first = got
        assert torch.equal(got, first)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,past", [(1, 77), (5, 60), (150, 0), (150, 70)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(dim, new, past):
    dtype, n = torch.bfloat16, new + past
    b = ref.Batch([new, 1], [n, 33], 2, dim, 16, dtype)
    at = n - 1 - new // 2  # one of the new tokens (the only one of a single row)
    b.value.view(-1, 2, dim)[b.slots[0][at], 0, 3] = torch.nan
    b.value.view(-1, 2, dim)[b.slots[0][at], 1, 5] = torch.inf
    q = _q(b, 4, dim, dtype)
    got = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=new, scale=0.1)
    row = at - past  # rows from here on see it
    assert torch.isnan(got[row:new, :2, 3]).all() and (got[row:new, 2:, 5] == torch.inf).all()
    fin = got.clone()
    fin[row:new, :2, 3] = 0
    fin[row:new, 2:, 5] = 0
    assert torch.isfinite(fin).all()
    want, _, mag, smax = ref.attention(q, b.k_of, b.v_of, b.starts, b.lens, 0.1, 0)
    want = torch.where(torch.isfinite(want), want, 0.0)
    assert ((fin.double() - want).abs() <= ref.attention_tolerance(dtype, dtype, mag, smax, dim, n)).all()


def test_scores_of_any_size():
    # large scores of both signs: one key takes all; all keys equal; -inf scores count for nothing
    b = ref.Batch([1, 4, 130], [500, 500, 600], 1, 128, 16, torch.bfloat16)
    q = _q(b, 2, 128, torch.bfloat16, amp=40.0)
    for scale in (1.0, -1.0, 0.0):
        got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=130,
                                      scale=scale, return_lse=True)
        _check(got, lse, b, q, scale, 0)


def test_many_short_sequences():
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(1, 90, (700,), generator=g).tolist()
    b = ref.Batch([1] * 700, lens, 1, 64, 16, torch.float16)
    q = _q(b, 2, 64, torch.float16)
    got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=1, scale=0.125,
                                  return_lse=True)
    _check(got, lse, b, q, 0.125, 0)


def test_same_result_on_any_stream_in_a_graph_and_twice_at_once():
    b = ref.Batch([1, 1, 1, 1], [900, 17, 3000, 1], 2, 256, 16, torch.bfloat16)
    q = _q(b, 8, 256, torch.bfloat16)

    def call(x=q):
        return hk.paged_attention(x, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=1, scale=0.0625)

    first = call()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for i in range(10):
        for s, x in ((s1, q), (s2, -q)):
            with torch.cuda.stream(s):
                outs.append((x is q, call(x)))
    torch.cuda.synchronize()
    minus = call(-q)
    assert all(torch.equal(o, first if same else minus) for same, o in outs)
    graph, x = torch.cuda.CUDAGraph(), q.clone()
    with torch.cuda.graph(graph):
        y = call(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    # the graph follows the lengths
    b.kv_lens.copy_(torch.tensor([1000 - 150, 5, 2222, 1], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    b.lens = [850, 5, 2222, 1]
    b.slots = [s[:n] for s, n in zip(b.slots, b.lens)]
    _check(y, None, b, q, 0.0625, 0)


def test_empty_calls():
    b = ref.Batch([], [], 2, 64, 16, torch.float16)
    q = torch.empty((0, 4, 64), dtype=torch.float16, device="cuda")
    assert hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=0,
                              scale=1.0).shape == (0, 4, 64)
    k = torch.empty((0, 2, 64), dtype=torch.float16, device="cuda")
    assert hk.prompt_attention(q, k, k, b.query_starts, max_query_len=0, scale=1.0).shape == (0, 4, 64)
    assert hk.paged_kv_append(k, k, b.key, b.value, b.table, b.query_starts, b.kv_lens, q=q).shape == (0, 4, 64)


@pytest.mark.parametrize("dim,rot_half,in_dtype,dtype,heads,kv_heads,norm,page", [
    (64, 32, torch.float32, torch.float16, 4, 4, False, 16),
    (64, 10, torch.bfloat16, torch.bfloat16, 4, 1, True, 64),
    (128, 32, torch.float32, torch.bfloat16, 32, 8, False, 16),
    (128, 64, torch.float16, torch.float16, 7, 1, True, 32),
    (256, 128, torch.float32, torch.float16, 8, 2, True, 16),
    (256, 0, torch.float32, torch.bfloat16, 40, 8, True, 256),
    (256, 64, torch.bfloat16, torch.bfloat16, 2, 2, False, 128),
])
def test_append(dim, rot_half, in_dtype, dtype, heads, kv_heads, norm, page):
    new = [1, 0, 37, 5, 1, 130, 4]
    lens = [1, 20, 37, 500, 1000, 140, 2]  # the last sequence: two rows before its first key
    b = ref.Batch(new, lens, kv_heads, dim, page, dtype, spare_rows=4)
    kc, vc = b.key.clone(), b.value.clone()
    x = (torch.randn((b.rows, heads + 2 * kv_heads, dim), device="cuda", generator=b.gen) * 2).to(in_dtype)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    inv = 1e6 ** (-torch.arange(rot_half, dtype=torch.float64, device="cuda") / max(1, rot_half))
    qw, kw = (1 + 0.2 * torch.randn(dim, device="cuda", generator=b.gen) for _ in range(2))
    q_out = torch.full((b.rows, heads, dim), 7.0, dtype=dtype, device="cuda")
    got = hk.paged_kv_append(k, v, kc, vc, b.table, b.query_starts, b.kv_lens, q=q, inv_freq=inv if rot_half else None,
                             q_norm=qw if norm else None, k_norm=kw if norm else None, norm_v=norm, eps=1e-5,
                             q_out=q_out)
    assert got is q_out
    seq, pos = ref.positions(b.starts, lens, b.rows, "cuda")
    live = pos >= 0
    qd, kd, vd = q.double(), k.double(), v.double()
    if norm:
        qd, kd, vd = ref.rms(qd, qw, 1e-5), ref.rms(kd, kw, 1e-5), ref.rms(vd, None, 1e-5)
    qr, kr = ref.rotate(qd, pos, inv), ref.rotate(kd, pos, inv)

    def near(a, want, full):
        # one rounding to the 16-bit type; norm, angle and the two products of
        # the rotation in f32 (a dozen roundings of 2^-24 and the angle's 2^-22
        # against the size of the pair, at most sqrt(2) of the row's largest)
        tol = torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + 2.0 ** -19 * full.abs().amax(-1, keepdim=True)
        assert ((a.double() - want).abs() <= tol).all()

    near(q_out[live], qr[live], qd[live])
    assert (q_out[~live] == 7.0).all()
    slot = torch.stack([b.slots[s][p] for s, p in zip(seq[live].tolist(), pos[live].tolist())])
    near(kc.view(-1, kv_heads, dim)[slot], kr[live], kd[live])
    near(vc.view(-1, kv_heads, dim)[slot], vd[live], vd[live])
    # nothing else was written
    other = torch.ones(kc.shape[0] * page, dtype=torch.bool, device="cuda")
    other[slot] = False
    for c, was in ((kc, b.key), (vc, b.value)):
        a, w = (t.view(-1, kv_heads, dim)[other].view(torch.int16) for t in (c, was))
        assert torch.equal(a, w)


def test_append_far_positions():
    # the angle keeps its precision where f32 would have lost it
    dim, pos = 64, 1_500_000_003
    inv = torch.tensor([1.0, 0.5, 0.1, 1e-9] * 8, dtype=torch.float64, device="cuda")
    k = torch.randn((1, 1, dim), device="cuda")
    kc = torch.zeros((1, 1024, 1, dim), dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.zeros((1, pos // 1024 + 1), dtype=torch.int32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    hk.paged_kv_append(k, k, kc, vc, table, torch.tensor([0, 1], **i32), torch.tensor([pos + 1], **i32), inv_freq=inv)
    want = ref.rotate(k.double(), torch.tensor([pos], device="cuda"), inv)[0, 0]
    assert ((kc[0, pos % 1024, 0].double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -18).all()


def test_cache_of_more_than_32_bits_of_bytes():
    pages, page, kv_heads, dim = 70_000, 64, 8, 128  # 9.2 GB of keys
    key = torch.empty((pages, page, kv_heads, dim), dtype=torch.float16, device="cuda")
    value = torch.empty_like(key)
    own = [pages - 1, 0, pages - 2, 33_000]
    n = 4 * page - 3
    x = torch.randn((n, 2 * kv_heads, dim), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([own], **i32)
    hk.paged_kv_append(x[:, :kv_heads], x[:, kv_heads:], key, value, table, torch.tensor([0, n], **i32),
                       torch.tensor([n], **i32))
    q = torch.randn((3, kv_heads, dim), device="cuda").half()
    got = hk.paged_attention(q, key, value, table, torch.tensor([0, 3], **i32), torch.tensor([n], **i32),
                             max_query_len=3, scale=0.1)
    k, v = x[:, :kv_heads].half(), x[:, kv_heads:].half()
    want, _, mag, smax = ref.attention(q, lambda s: k, lambda s: v, [0, 3], [n], 0.1, 0)
    assert ((got.double() - want).abs() <= ref.attention_tolerance(q.dtype, q.dtype, mag, smax, dim, n)).all()


def test_pages_outside_the_cache_are_reported():
    b = ref.Batch([1, 1], [100, 40], 2, 64, 16, torch.float16)
    q = _q(b, 4, 64, torch.float16)
    hk.device_error()
    for entry in (-1, b.key.shape[0], 2 ** 31 - 1):
        t = b.table.clone()
        t[0, 2] = entry
        hk.paged_attention(q, b.key, b.value, t, b.query_starts, b.kv_lens, max_query_len=1, scale=0.1)
        with pytest.raises(hk.CudaKernelError) as e:
            hk.device_error()
        assert e.value.code == hk.ERR_SHAPE
        t = b.table.clone()
        t[0, 6] = entry  # the page of the new token
        kc, vc = b.key.clone(), b.value.clone()
        x = torch.randn((2, 2, 64), device="cuda")
        hk.paged_kv_append(x, x, kc, vc, t, b.query_starts, b.kv_lens)
        with pytest.raises(hk.CudaKernelError):
            hk.device_error()
        assert torch.equal(kc.view(-1, 2, 64)[b.slots[0]], b.k_of(0))
        assert torch.equal(kc.view(-1, 2, 64)[b.slots[1][-1]], x[1].half())
    for lens in ([100_000, 40], [-5, 40]):
        hk.paged_attention(q, b.key, b.value, b.table[:, :7].contiguous(), b.query_starts,
                           torch.tensor(lens, dtype=torch.int32, device="cuda"), max_query_len=1, scale=0.1)
        with pytest.raises(hk.CudaKernelError):
            hk.device_error()
    for starts in ([0, 1, 9], [-3, 1, 2], [0, 2, 1]):
        hk.paged_attention(q, b.key, b.value, b.table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                           b.kv_lens, max_query_len=1, scale=0.1)
        with pytest.raises(hk.CudaKernelError):
            hk.device_error()
    got = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=1, scale=0.1)
    hk.device_error()
    _check(got, None, b, q, 0.1, 0)
