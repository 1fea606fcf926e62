"""Penalties, biases, masks and the top-k over logits against the definition
in 64 bits: the values are f64 results rounded once, so ids and values are
equal, not merely near."""
import numpy as np
import pytest
import torch

from heliopause_b200 import kernels as hk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    hk.init_device(0)


def reference(logits, k, hist=None, prompt=None, rep=None, freq=None, pres=None, bias=None, allowed=None):
    rows, vocab = logits.shape
    ids, vals = np.full((rows, k), -1, np.int32), np.full((rows, k), -np.inf, np.float32)
    for r in range(rows):
        x = logits[r].astype(np.float64)
        if hist is not None:
            h = np.asarray(hist[r], np.int64)
            live = (h >= 0) & (h < vocab)
            out = np.arange(len(h)) >= (prompt[r] if prompt is not None else 0)
            seen = np.zeros(vocab, bool)
            seen[h[live]] = True
            count = np.bincount(h[live & out], minlength=vocab)
            if rep is not None:
                x = np.where(seen, np.where(x > 0, x / np.float64(rep[r]), x * np.float64(rep[r])), x)
            f = np.float64(freq[r]) if freq is not None else 0.0
            p = np.float64(pres[r]) if pres is not None else 0.0
            x = np.where(count > 0, x - f * count - p, x)
        if bias is not None:
            for i, b in bias[r]:
                if 0 <= i < vocab:
                    x[i] += 0.0
            add, has = np.zeros(vocab), np.zeros(vocab, bool)
            for i, b in bias[r]:
                if 0 <= i < vocab:
                    add[i] += np.float64(np.float32(b))
                    has[i] = True
            x = np.where(has, x + add, x)
        x = x.astype(np.float32)
        if allowed is not None:
            x = np.where(allowed[r], x, np.float32(-np.inf))
        live = np.nonzero(x > -np.inf)[0]  # NaN and -inf are no candidates
        order = live[np.argsort(-x[live], kind="stable")][:k]
        ids[r, :len(order)], vals[r, :len(order)] = order, x[order]
    return ids, vals


def _lists(xs, dtype):
    starts = np.concatenate([[0], np.cumsum([len(x) for x in xs])])
    flat = np.concatenate([np.asarray(x, np.float64) for x in xs]) if len(xs) else np.zeros(0)
    return torch.tensor(flat, dtype=dtype, device="cuda"), torch.tensor(starts, dtype=torch.int32, device="cuda")


def _run(logits, k, hist=None, prompt=None, rep=None, freq=None, pres=None, bias=None, allowed=None, stride=0):
    rows, vocab = logits.shape
    x = torch.full((rows, vocab + stride), 1e30, device="cuda")
    x[:, :vocab] = torch.from_numpy(logits)
    kw = {}
    if hist is not None:
        kw["history"], kw["history_starts"] = _lists(hist, torch.int32)
    if prompt is not None:
        kw["prompt_lens"] = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    for n, v in (("repetition", rep), ("frequency", freq), ("presence", pres)):
        if v is not None:
            kw[n] = torch.tensor(v, dtype=torch.float32, device="cuda")
    if bias is not None:
        kw["bias_ids"], kw["bias_starts"] = _lists([[i for i, _ in b] for b in bias], torch.int32)
        kw["bias_values"] = _lists([[v for _, v in b] for b in bias], torch.float32)[0]
    if allowed is not None:
        words = np.zeros((rows, (vocab + 31) // 32 + 1, 32), np.uint64)
        words.reshape(rows, -1)[:, :vocab] = allowed
        packed = (words << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)
        kw["allowed"] = torch.from_numpy(packed).cuda()
    ids, vals = hk.logits_topk(x[:, :vocab], k, **kw)
    return ids.cpu().numpy(), vals.cpu().numpy()


def _same(logits, k, stride=0, **kw):
    got, want = _run(logits, k, stride=stride, **kw), reference(logits, k, **kw)
    assert np.array_equal(got[0], want[0])
    assert np.array_equal(got[1], want[1])


@pytest.mark.parametrize("rows,vocab,k,stride", [
    (1, 1, 1, 0), (1, 64, 64, 0), (3, 4095, 7, 0), (2, 4096, 64, 0), (2, 4097, 64, 3), (5, 32003, 40, 1),
    (1, 262144, 64, 0), (4, 100_003, 1, 0), (70, 5000, 20, 0), (1, 1 << 20, 64, 0),
])
def test_plain_topk(rows, vocab, k, stride):
    g = np.random.default_rng(vocab)
    _same((g.standard_normal((rows, vocab)) * 3).astype(np.float32), k, stride=stride)


@pytest.mark.parametrize("rows,vocab,k,hist", [(1, 300, 40, 50), (6, 9001, 64, 3000), (3, 262144, 64, 5000)])
def test_everything_at_once(rows, vocab, k, hist):
    g = np.random.default_rng(hist)
    x = (g.standard_normal((rows, vocab)) * 3).astype(np.float32)
    hs = [g.choice(g.integers(-2, vocab + 2, max(2, hist // 3)), g.integers(0, hist + 1)) for _ in range(rows)]
    f = lambda lo, hi: g.uniform(lo, hi, rows).astype(np.float32)  # noqa: E731
    top = np.argsort(-x, axis=1)[:, :30]
    bias = [[(int(i), float(v)) for i, v in zip(np.concatenate([g.choice(top[r], 20), g.integers(-1, vocab + 1, 30)]),
                                                g.standard_normal(50) * 4)] for r in range(rows)]
    _same(x, k, hist=hs, prompt=g.integers(0, hist // 2, rows), rep=f(0.7, 1.6), freq=f(-0.5, 1), pres=f(-1, 1), bias=bias,
          allowed=g.random((rows, vocab)) < 0.4)


def test_each_part_alone():
    g = np.random.default_rng(5)
    x = (g.standard_normal((3, 6000)) * 2).astype(np.float32)
    hs = [g.choice(np.argsort(-x[r])[:100], 400) for r in range(3)]
    one = np.array([1.3, 0.8, 1.0], np.float32)
    _same(x, 50, hist=hs, rep=one)
    _same(x, 50, hist=hs, freq=one)
    _same(x, 50, hist=hs, pres=one, prompt=np.array([0, 400, 1000]))
    _same(x, 50, hist=hs)
    _same(x, 50, bias=[[(7, 30.0), (7, -31.0), (8, 5.0)], [], [(5999, 9.0)] * 70])
    _same(x, 50, allowed=np.arange(6000)[None] % np.array([1, 7, 997])[:, None] == 0)


def test_values_at_the_edges():
    k, vocab = 16, 9000
    x = np.full((9, vocab), -np.inf, np.float32)
    x[1, 5000] = 3.0                          # one candidate
    x[2] = 0.0
    x[2, ::2] = -0.0                          # both zeros are one value: ties by id
    x[3] = 2.5                                # all equal
    x[4] = np.nan
    x[4, 17] = -1.0                           # NaN is no candidate
    x[5] = 1.0
    x[5, 8999] = np.inf
    x[6] = np.finfo(np.float32).min           # the lowest finite value is one
    x[7] = np.arange(vocab)                   # ascending, and descending
    x[8] = -np.arange(vocab)
    _same(x, k)
    _same(x, 64)
    _same(x, k, bias=[[(3, 1.0)], [(5000, -np.inf)], [(9, np.inf)], [], [(17, np.nan)], [(8999, -np.inf)], [], [], []])
    _same(x, k, allowed=np.zeros((9, vocab), bool))


def test_ties_across_chunks_and_many_equal_values():
    g = np.random.default_rng(8)
    _same(g.integers(-3, 3, (4, 50_000)).astype(np.float32), 64)
    _same(g.integers(-1000, 1000, (4, 50_000)).astype(np.float32), 64)


def test_ties_between_touched_and_untouched_tokens():
    # integer logits: penalties and biases put touched tokens on the values of
    # untouched ones, behind and before them
    g = np.random.default_rng(21)
    rows, vocab = 3, 40_000
    x = g.integers(-4, 5, (rows, vocab)).astype(np.float32)
    x[:, g.choice(vocab, 300, replace=False)] = 9.0
    hs = [np.concatenate([g.integers(0, vocab, 500), np.nonzero(x[r] == 9)[0][-60:]]) for r in range(rows)]
    bias = [[(int(i), 5.0) for i in np.concatenate([g.choice(np.nonzero(x[r] == 4)[0], 100), [vocab - 1, 0]])] for r in range(rows)]
    for k in (5, 64):
        _same(x, k, hist=hs, freq=np.ones(rows, np.float32), bias=bias)
        _same(x, k, hist=hs, freq=-np.ones(rows, np.float32), bias=bias, allowed=g.random((rows, vocab)) < 0.5)


def test_long_histories_and_many_biases():
    # more tokens than a count's bits, more biases and listed tokens than the lists hold
    g = np.random.default_rng(22)
    x = (g.standard_normal((2, 70_000)) * 2).astype(np.float32)
    hs = [np.full(20_000, 77), g.integers(0, 12_000, 30_000)]
    bias = [[(int(i), float(v)) for i, v in zip(g.integers(0, 9000, 1500), g.standard_normal(1500))], [(5, 1.5)] * 700]
    _same(x, 64, hist=hs, prompt=np.array([10, 5000]), rep=np.array([1.1, 0.9], np.float32),
          freq=np.array([-0.001, 0.25], np.float32), pres=np.array([0.5, -0.5], np.float32), bias=bias)


def test_starts_outside_the_lists_are_bounded():
    x = torch.randn((2, 500), device="cuda")
    h = torch.arange(10, dtype=torch.int32, device="cuda")
    one = torch.full((2,), 2.0, device="cuda")
    for starts in ([-5, 4, 10**9], [8, 3, 2], [0, 10, 10]):
        a = np.clip(starts, 0, 10)
        hs = [list(range(a[r], max(a[r], a[r + 1]))) for r in range(2)]
        ids, vals = hk.logits_topk(x, 20, history=h, history_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                   frequency=one)
        want = reference(x.cpu().numpy(), 20, hist=hs, freq=[2.0, 2.0])
        assert np.array_equal(ids.cpu().numpy(), want[0]) and np.array_equal(vals.cpu().numpy(), want[1])


def test_streams_graph_and_the_sampler():
    g = np.random.default_rng(11)
    x = torch.from_numpy((g.standard_normal((4, 30_000)) * 3).astype(np.float32)).cuda()
    first = hk.logits_topk(x, 40)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((i % 2, hk.logits_topk(x if i % 2 else -x, 40)))
    torch.cuda.synchronize()
    minus = hk.logits_topk(-x, 40)
    for same, (ids, vals) in outs:
        want = first if same else minus
        assert torch.equal(ids, want[0]) and torch.equal(vals, want[1])
    graph, y = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        ids, vals = hk.logits_topk(y, 40)
    y.copy_(-x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ids, minus[0]) and torch.equal(vals, minus[1])
    # a row whose grammar leaves two tokens: the sampler draws one of them
    allowed = torch.zeros((4, 938), dtype=torch.int32, device="cuda")
    allowed[:, 3] = 0b101  # tokens 96 and 98
    ids, vals = hk.logits_topk(x, 8, allowed=allowed)
    assert sorted(ids[0, :2].tolist()) == [96, 98] and (ids[0, 2:] == -1).all()
    token = torch.empty(1, dtype=torch.int32, device="cuda")
    for seed in range(20):
        hk.sample_candidates(ids[0], vals[0], top_k=8, top_p=0.95, temperature=1.0, greedy=False, rng_state=seed,
                             token_out=token)
        assert token.item() in (96, 98)
