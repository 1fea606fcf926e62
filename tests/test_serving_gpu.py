"""The serving operators together, as a batch of chats uses them, and attention
whose keys are summed in parts -- against plain 64-bit forms."""
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
    hk.device_error()  # no batch here points outside its buffers


@pytest.mark.parametrize("dim,dtype,heads,kv_heads,page,new,lens,window,scale", [
    (256, torch.bfloat16, 8, 2, 64, [100], [5000], 0, 1.0),
    (256, torch.float16, 8, 2, 16, [9, 100, 40, 0], [1030, 4100, 40, 70], 0, -1.0),  # below and above 8 tiles
    (256, torch.bfloat16, 9, 1, 128, [64], [3001], 2100, 1.0),
    (128, torch.float16, 32, 8, 64, [70, 33], [4100, 2049], 0, 1.0),
    (128, torch.bfloat16, 14, 2, 16, [50], [6001], 0, 1.0),    # a group that does not divide a tile's rows
    (128, torch.bfloat16, 6, 2, 1024, [131], [2500], 1500, -1.0),
    (64, torch.float16, 4, 4, 32, [33, 300], [2047, 5555], 0, 1.0),
    (64, torch.bfloat16, 24, 2, 64, [12] * 3, [1024, 8200, 3333], 0, 1.0),
    (64, torch.bfloat16, 128, 1, 64, [2], [4999], 4000, 1.0),
])
@pytest.mark.parametrize("out32", [False, True])
def test_keys_in_parts(dim, dtype, heads, kv_heads, page, new, lens, window, scale, out32):
    b = ref.Batch(new, lens, kv_heads, dim, page, dtype, spare_rows=2)
    q = _q(b, heads, dim, dtype, strided=True)
    ot = torch.float32 if out32 else dtype
    out = torch.full((b.rows, heads, dim), 7.0, dtype=ot, device="cuda")
    sc = scale * dim ** -0.5
    _, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(new),
                                scale=sc, window=window, out=out, return_lse=True)
    assert (out[b.starts[-1]:] == 7.0).all()
    _check(out, lse, b, q, sc, window, ot)
    again = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(new),
                               scale=sc, window=window, out_dtype=ot)
    assert torch.equal(again[:b.starts[-1]], out[:b.starts[-1]])  # parts are joined in one order


@pytest.mark.parametrize("dim,dtype,heads,kv_heads,new,window", [
    (256, torch.float16, 2, 1, [4000], 0),
    (128, torch.bfloat16, 4, 1, [3, 3000, 500], 0),
    (64, torch.float16, 7, 1, [1, 2600], 1700),
])
def test_one_long_prompt_in_parts(dim, dtype, heads, kv_heads, new, window):
    b = ref.Batch(new, new, kv_heads, dim, 16, dtype)
    k = torch.cat([b.k_of(s) for s in range(len(new))])
    v = torch.cat([b.v_of(s) for s in range(len(new))])
    q = _q(b, heads, dim, dtype)
    got, lse = hk.prompt_attention(q, k, v, b.query_starts, max_query_len=max(new), scale=dim ** -0.5, window=window,
                                   return_lse=True)
    _check(got, lse, b, q, dim ** -0.5, window)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1100])
def test_values_that_are_not_finite_in_parts(dim, window):
    # seen by every row, by some rows, and (with the window) only by the first rows
    new, n, dtype = 100, 3000, torch.bfloat16
    b = ref.Batch([new], [n], 1, dim, 64, dtype)
    past = n - new
    v = b.value.view(-1, 1, dim)
    spots = [(n - 30, 1, torch.nan), (n - 60, 2, torch.inf)]
    spots.append((past - 1100 + 40, 4, torch.nan) if window else (700, 4, torch.inf))
    for j, d, x in spots:
        v[b.slots[0][j], 0, d] = x
    q = _q(b, 4, dim, dtype)
    got = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=new, scale=0.05,
                             window=window)
    pos = torch.arange(past, n, device="cuda")
    fin = got.clone()
    for j, d, x in spots:
        sees = (pos >= j) & ((pos - j < window) if window else (pos >= 0))
        assert 0 < sees.sum() <= new
        hit = got[sees][:, :, d]
        assert torch.isnan(hit).all() if x != x else (hit == x).all()
        fin[sees.nonzero()[:, 0], :, d] = 0
    assert torch.isfinite(fin).all()
    want, _, mag, smax = ref.attention(q, b.k_of, b.v_of, b.starts, b.lens, 0.05, window)
    keep = torch.isfinite(want)
    d = (fin.double() - torch.where(keep, want, 0.0)).abs()
    tol = ref.attention_tolerance(dtype, dtype, mag, smax, dim, n)
    assert (d <= tol)[keep].all()


def test_parts_on_two_streams_and_in_a_graph():
    b = ref.Batch([128], [6000], 2, 256, 64, torch.float16)
    c = ref.Batch([60, 80], [3000, 4000], 8, 128, 16, torch.bfloat16, seed=1)
    qb, qc = _q(b, 8, 256, torch.float16), _q(c, 32, 128, torch.bfloat16)

    def one(x, q):
        return hk.paged_attention(q, x.key, x.value, x.table, x.query_starts, x.kv_lens, max_query_len=128, scale=0.06)

    want_b, want_c = one(b, qb), one(c, qc)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):  # both at once, each with a workspace of its own
        with torch.cuda.stream(s1):
            got.append((one(b, qb), want_b))
        with torch.cuda.stream(s2):
            got.append((one(c, qc), want_c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [one(b, qb), one(c, qc), one(b, qb)]
    for _ in range(3):
        for o in outs:
            o.zero_()
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want_b) and torch.equal(outs[1], want_c) and torch.equal(outs[2], want_b)


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 200, 1), (128, 257, 1), (256, 96, 1), (64, 1024, 1)])
@pytest.mark.parametrize("window", [0, 2 ** 31 - 1])
def test_wide_groups_and_rows_of_no_token(dim, heads, kv_heads, window):
    # groups around and above a tile's 128 rows, a window wider than any length, and
    # query rows behind the last sequence that hold NaN and infinities
    b = ref.Batch([3, 2, 0, 5], [3, 1500, 7, 70], kv_heads, dim, 32, torch.bfloat16, spare_rows=9)
    q = _q(b, heads, dim, torch.bfloat16)
    q[b.starts[-1]:] = torch.tensor([torch.nan, torch.inf, -torch.inf] * 3, device="cuda").view(9, 1, 1)
    out = torch.full((b.rows, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    _, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=5,
                                scale=dim ** -0.5, window=window, out=out, return_lse=True)
    assert (out[b.starts[-1]:] == 7.0).all() and (lse[b.starts[-1]:] == -torch.inf).all()
    n = b.starts[-1]
    c = b.query_starts.clone()
    _check(out[:n], lse[:n], b, q[:n], dim ** -0.5, 0)
    assert torch.equal(c, b.query_starts)


@pytest.mark.parametrize("dim,heads", [(256, 12), (128, 8), (64, 4)])
def test_many_sequences_in_parts(dim, heads):
    # more sequences than one look at their lengths takes in, some of them empty,
    # and few enough items that the long ones are cut into parts
    new = [20 + i % 3 if i % 5 else 0 for i in range(43)]
    lens = [max(n, (i * 977) % 2900) for i, n in enumerate(new)]
    b = ref.Batch(new, lens, 1, dim, 16, torch.bfloat16, spare_rows=1)
    q = _q(b, heads, dim, torch.bfloat16)
    got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=max(new),
                                  scale=dim ** -0.5, return_lse=True)
    _check(got, lse, b, q, dim ** -0.5, 0)


@pytest.mark.parametrize("hint", [1, 3, 40, 10 ** 6])
def test_any_most_new_tokens_gives_the_same_rows(hint):
    # max_query_len chooses the kernel, not the result
    b = ref.Batch([40, 1, 7], [2100, 900, 7], 2, 128, 16, torch.float16)
    q = _q(b, 8, 128, torch.float16)
    got, lse = hk.paged_attention(q, b.key, b.value, b.table, b.query_starts, b.kv_lens, max_query_len=hint,
                                  scale=0.08, return_lse=True)
    _check(got, lse, b, q, 0.08, 0)


@pytest.mark.parametrize("dim,heads,kv_heads,dtype", [(256, 8, 2, torch.float16), (64, 6, 3, torch.bfloat16)])
def test_a_batch_of_chats(dim, heads, kv_heads, dtype):
    """Prompts, decode steps and a verify step of four chats through a cache,
    then the penalised logits' best tokens and the sampler: every step's
    attention against 64-bit attention over all the keys so far, and the tokens
    against the plain forms."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    page, width, vocab, hidden = 16, 24, 5003, 192
    new0 = [37, 1, 300, 129]
    seqs = len(new0)
    order = torch.randperm(seqs * width, generator=torch.Generator().manual_seed(1)).int()
    table = order.view(seqs, width).cuda()
    key = torch.full((seqs * width, page, kv_heads, dim), torch.nan, dtype=dtype, device="cuda")
    value = torch.full_like(key, torch.nan)
    inv = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device="cuda") / (dim // 2))
    qn, kn = (torch.rand(dim, device="cuda", generator=gen) + 0.5 for _ in range(2))
    rnd = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    wqkv = rnd(hidden, (heads + 2 * kv_heads) * dim) * hidden ** -0.5
    head = rnd(heads * dim, vocab) * (heads * dim) ** -0.5
    lens = [0] * seqs
    ks, vs = [None] * seqs, [None] * seqs  # the caches' rows so far, packed
    hist = [[] for _ in range(seqs)]
    scale = dim ** -0.5
    for step, new in enumerate([new0, [1] * seqs, [5, 0, 5, 5], [1] * seqs]):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        lens = [a + n for a, n in zip(lens, new)]
        rows = starts[-1]
        qs = torch.tensor(starts, dtype=torch.int32, device="cuda")
        kl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        x = rnd(rows, hidden)
        qkv = (x @ wqkv).view(rows, heads + 2 * kv_heads, dim)  # heads of one projection: strided views
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
        qr = hk.paged_kv_append(k, v, key, value, table, qs, kl, q=q, inv_freq=inv, q_norm=qn, k_norm=kn, norm_v=True)
        flat_k, flat_v = key.view(-1, kv_heads, dim), value.view(-1, kv_heads, dim)
        for s in range(seqs):
            j = torch.arange(lens[s], device="cuda")
            slot = table[s].long()[j // page] * page + j % page
            nk, nv = flat_k[slot], flat_v[slot]
            assert torch.isfinite(nk).all() and torch.isfinite(nv).all()
            if ks[s] is not None:  # what was there stays
                assert torch.equal(nk[:ks[s].shape[0]], ks[s]) and torch.equal(nv[:vs[s].shape[0]], vs[s])
            ks[s], vs[s] = nk, nv
        got = hk.paged_attention(qr, key, value, table, qs, kl, max_query_len=max(new), scale=scale)
        want, _, mag, smax = ref.attention(qr, lambda s: ks[s], lambda s: vs[s], starts, lens, scale, 0)
        tol = ref.attention_tolerance(dtype, dtype, mag, smax, dim, max(lens))
        assert ((got.double() - want).abs() <= tol).all()
        if step == 0:  # the prompts' own rows, without the cache
            again = hk.prompt_attention(qr, torch.cat(ks), torch.cat(vs), qs, max_query_len=max(new), scale=scale)
            assert ((again.double() - want).abs() <= tol).all()
        last = torch.tensor([max(e - 1, 0) for e in starts[1:]], device="cuda")
        logits = got[last].float().view(seqs, -1) @ head
        hs = [0]
        for h in hist:
            hs.append(hs[-1] + len(h))
        i32 = lambda y: torch.tensor(y, dtype=torch.int32, device="cuda")  # noqa: E731
        f32 = lambda y: torch.tensor(y, dtype=torch.float32, device="cuda")  # noqa: E731
        flat = [t for h in hist for t in h]
        kept = logits.clone()
        ids, vals = hk.logits_topk(logits, 40, history=i32(flat), history_starts=i32(hs), prompt_lens=i32([0] * seqs),
                                   repetition=f32([1.5] * seqs), frequency=f32([0.25] * seqs),
                                   presence=f32([0.5] * seqs))
        assert torch.equal(logits, kept)
        token = torch.empty(1, dtype=torch.int32, device="cuda")
        for s in range(seqs):
            plain = kept[s].cpu().double()
            for t in set(hist[s]):
                plain[t] = plain[t] / 1.5 if plain[t] > 0 else plain[t] * 1.5
                plain[t] -= 0.25 * hist[s].count(t) + 0.5
            got_v = vals[s].cpu().double()
            # each of the (at most four) f32 steps rounds by 2^-24 of what it gives
            near = lambda a, b: (a - b).abs() <= 4 * 2.0 ** -24 * (a.abs() + b.abs() + 2.0)  # noqa: E731
            assert near(got_v, plain[ids[s].cpu().long()]).all()
            assert near(got_v, plain.sort(descending=True).values[:40]).all()
            hk.sample_candidates(ids[s], vals[s], top_k=40, top_p=0.9, temperature=0.8, greedy=step == 3, rng_state=step,
                                 token_out=token)
            hist[s].append(int(token))
            assert hist[s][-1] in ids[s].tolist() and (step < 3 or hist[s][-1] == int(ids[s, 0]))


class _NothingPlain:
    """Stands in for the host module: every call goes the whole way in Python."""

    def __getattr__(self, name):
        return lambda *a: NotImplemented


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_both_host_paths_make_the_same_calls(monkeypatch, dtype):
    b = ref.Batch([40, 1, 0, 7], [340, 9, 3, 7], 2, 128, 16, dtype, spare_rows=2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    inv = torch.rand(32, device="cuda", dtype=torch.float64, generator=gen)
    norm = torch.rand(128, device="cuda", generator=gen)
    x = rnd(b.rows, 12, 128)
    logits = rnd(3, 7001)
    i32 = lambda y: torch.tensor(y, dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda y: torch.tensor(y, dtype=torch.float32, device="cuda")  # noqa: E731
    full = dict(history=i32([5, 6, 6, 9]), history_starts=i32([0, 3, 3, 4]), prompt_lens=i32([1, 0, 0]),
                repetition=f32([1.5, 1, 2]), frequency=f32([0.5, 0, 0]), presence=f32([0.1, 0, 0]),
                bias_ids=i32([7, 8]), bias_values=f32([3.0, -2.0]), bias_starts=i32([0, 1, 1, 2]),
                allowed=torch.randint(-2 ** 31, 2 ** 31 - 1, (3, 220), dtype=torch.int32, device="cuda", generator=gen))

    def run():
        key, value = b.key.clone(), b.value.clone()
        res = []
        for q, kn, freq in ((x[:, :8], norm, inv), (None, None, None), (x[:, :8], None, inv)):
            out = torch.zeros((b.rows, 8, 128), dtype=dtype, device="cuda") if q is not None else None
            r = hk.paged_kv_append(x[:, 8:10], x[:, 10:], key, value, b.table, b.query_starts, b.kv_lens, q=q, inv_freq=freq,
                                   q_norm=kn, k_norm=kn, norm_v=q is not None, q_out=out)
            assert r is out
            res += [key.clone(), value.clone()] + ([r] if r is not None else [])
        q = x[:, :8].to(dtype)
        n = b.starts[-1]
        for kw in ({}, {"window": 5}, {"out_dtype": torch.float32}, {"out": torch.empty_like(q)}):
            got = hk.paged_attention(q, key, value, b.table, b.query_starts, b.kv_lens, max_query_len=40, scale=0.1, **kw)
            assert got is kw.get("out", got)
            res.append(got[:n].clone())
            k, v = x[:, 8:10].to(dtype), x[:, 10:].to(dtype)
            got = hk.prompt_attention(q, k, v, b.query_starts, max_query_len=40, scale=1, **kw)
            assert got is kw.get("out", got)
            res.append(got[:n].clone())
        for kw in ({}, full, {"allowed": full["allowed"]}):
            res += hk.logits_topk(logits, 17, **kw)
        res += hk.logits_topk(logits[:, 1:6001], 64)
        with pytest.raises(hk.CudaKernelError):
            hk.logits_topk(logits, 65)
        with pytest.raises(hk.CudaKernelError):
            hk.paged_attention(q, key, value, b.table.long(), b.query_starts, b.kv_lens, max_query_len=40, scale=0.1)
        with pytest.raises(hk.CudaKernelError):
            hk.prompt_attention(q, k, v[:1], b.query_starts, max_query_len=40, scale=0.1)
        with pytest.raises(hk.CudaKernelError):
            hk.paged_kv_append(x[:, 8:10], x[:, 10:], key, value, b.table, b.query_starts, b.kv_lens, k_norm=norm[:64])
        return res

    torch.manual_seed(0)
    fast = run()
    monkeypatch.setattr(hk, "_host", _NothingPlain())
    whole = run()
    assert len(fast) == len(whole)
    for a, c in zip(fast, whole):
        assert a.dtype == c.dtype and torch.equal(torch.nan_to_num(a.float(), 9.0), torch.nan_to_num(c.float(), 9.0))
