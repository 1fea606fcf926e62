"""The top-k over logits where a chunk of a row is a stream of 4 or 8 steps (many
rows of a large vocabulary): the floor that rises behind the third step, and
what it decides from.  Ids and values are equal to the definition's, and to
themselves from run to run."""
import numpy as np
import pytest
import torch

from heliopause_b200 import kernels as hk
from tests.test_logits_gpu import _run, _same, reference

pytestmark = pytest.mark.gpu

STEP = 4096       # tokens of a step
CHUNK = 8 * STEP  # of a chunk, where rows * ceil(vocab / CHUNK) >= 296


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    hk.init_device(0)


@pytest.mark.parametrize("rows,vocab,k", [(40, 262144, 1), (64, 151936, 1), (300, 32768, 1), (300, 32768, 2)])
def test_the_best_token_of_many_rows(rows, vocab, k):
    # few keys pass the first floor, so a chunk has kept about k of them when
    # it looks whether the floor can rise: the threads have to agree on it
    g = np.random.default_rng(vocab + k)
    x = (g.standard_normal((rows, vocab)) * 3).astype(np.float32)
    want = reference(x, k)
    d = torch.from_numpy(x).cuda()
    for _ in range(30):
        ids, vals = hk.logits_topk(d, k)
        assert np.array_equal(ids.cpu().numpy(), want[0]) and np.array_equal(vals.cpu().numpy(), want[1])


@pytest.mark.parametrize("rows,vocab,k", [(300, CHUNK, 1), (300, CHUNK, 40), (160, 2 * CHUNK - 77, 64)])
@pytest.mark.parametrize("touched", [False, True])
def test_masks_that_leave_about_k_tokens(rows, vocab, k, touched):
    # row r: k - 2 .. k + 2 tokens of the first three steps of every chunk, and up to
    # a hundred behind them, so that the number of kept keys crosses k there
    g = np.random.default_rng(k)
    x = (g.standard_normal((rows, vocab)) * 3).astype(np.float32)
    allowed = np.zeros((rows, vocab), bool)
    for r in range(rows):
        for c0 in range(0, vocab, CHUNK):
            early = g.choice(3 * STEP, max(0, k - 2 + r % 5), replace=False)
            late = 3 * STEP + g.choice(min(CHUNK, vocab - c0) - 3 * STEP, (0, 1, 3, 100)[r // 5 % 4], replace=False)
            allowed[r, c0 + np.concatenate([early, late])] = True
    kw = {}
    if touched:
        kw = dict(hist=[np.nonzero(allowed[r])[0][::3] for r in range(rows)], rep=np.full(rows, 1.25, np.float32),
                  freq=np.full(rows, 0.5, np.float32))
    want = reference(x, k, allowed=allowed, **kw)
    for _ in range(5):
        got = _run(x, k, allowed=allowed, **kw)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("rows,vocab,k,stride", [
    (20, 262144, 64, 0),       # 4 steps
    (40, 262144, 64, 0),       # 8 steps
    (100, 100_003, 40, 1),     # rows at odd addresses: single loads
    (150, CHUNK + 1, 64, 0),   # a chunk of one token
    (150, CHUNK + 6 * STEP + 5, 64, 3),
])
def test_streams_of_many_steps(rows, vocab, k, stride):
    g = np.random.default_rng(vocab)
    _same((g.standard_normal((rows, vocab)) * 3).astype(np.float32), k, stride=stride)


@pytest.mark.parametrize("k", [1, 5, 64])
def test_ties_across_the_rising_floor(k):
    # few distinct values, so that the floor is a value that later steps hold too;
    # penalties and biases put listed tokens on it, before and behind it
    g = np.random.default_rng(30 + k)
    rows, vocab = 300, CHUNK
    x = g.integers(-40, 41, (rows, vocab)).astype(np.float32)
    x[::3] = g.integers(-4000, 4001, (100, vocab))
    x[1::3] = np.where(g.random((100, vocab)) < 2e-3, 41.0, x[1::3])
    x[::2][x[::2] == 0] = -0.0
    _same(x, k)
    hs = [np.concatenate([g.integers(0, vocab, 200), np.argsort(-x[r], kind="stable")[:60]]) for r in range(rows)]
    bias = [[(int(i), float(v)) for i, v in zip(g.integers(0, vocab, 40), g.integers(-3, 45, 40))] for _ in range(rows)]
    _same(x, k, hist=hs, freq=np.ones(rows, np.float32), bias=bias)
    _same(x, k, hist=hs, freq=-np.ones(rows, np.float32), allowed=g.random((rows, vocab)) < 0.5)


def test_rows_that_overflow_the_kept_keys():
    # ascending rows keep every token, equal ones very many: the k best are then
    # found by passes over the chunk
    rows, vocab = 300, CHUNK
    x = np.tile(np.arange(vocab, dtype=np.float32), (rows, 1))
    x[1::4] = 1.5
    x[2::4] = x[2::4] // 64
    x[3::4, ::2] = -np.inf
    hs = [np.arange(vocab - 1 - r, vocab, 7) for r in range(rows)]
    _same(x, 64)
    _same(x, 64, hist=hs, rep=np.full(rows, 1.5, np.float32))


@pytest.mark.parametrize("distinct", [4095, 4096, 4097, 20_000])
def test_more_listed_tokens_than_the_list_holds(distinct):
    # of one chunk; and counts above the 14 bits of a token's counter
    g = np.random.default_rng(distinct)
    rows, vocab = 300, CHUNK
    x = (g.standard_normal((rows, vocab)) * 3).astype(np.float32)
    hs = [np.zeros(0, np.int64)] * rows
    hs[7] = np.tile(g.choice(vocab, distinct, replace=False), 2)
    hs[299] = np.concatenate([g.choice(vocab, distinct, replace=False), np.full(16_000, 11)])
    bias = [[]] * rows
    bias[299] = [(int(i), float(v)) for i, v in zip(g.integers(0, vocab, 600), g.standard_normal(600))]
    _same(x, 64, hist=hs, prompt=g.integers(0, 50, rows), rep=np.full(rows, 1.3, np.float32),
          freq=np.full(rows, 0.001, np.float32), pres=np.full(rows, 0.25, np.float32), bias=bias)


@pytest.mark.parametrize("k", [1, 64])
def test_edge_values_in_every_step(k):
    rows, vocab = 300, CHUNK
    g = np.random.default_rng(k)
    x = (g.standard_normal((rows, vocab)) * 3).astype(np.float32)
    for r in range(rows):
        at = r * 113 % vocab  # somewhere else in every row
        x[r, at:at + 9] = (np.inf, np.nan, -np.inf, np.finfo(np.float32).min, np.finfo(np.float32).max, -0.0, 0.0, 1e-45, -1e-45)[
            :vocab - at]
    x[5] = -np.inf
    x[6] = np.nan
    x[7] = -np.inf
    x[7, [3 * STEP, vocab - 1]] = 1.0
    x[8] = np.finfo(np.float32).min
    x[9] = np.where(np.arange(vocab) % 2, 1e-45, -1e-45)
    x[10] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    _same(x, k)
    _same(x, k, hist=[np.arange(r % 40) * 800 for r in range(rows)], pres=np.full(rows, 0.5, np.float32))
