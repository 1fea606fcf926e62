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
