"""Plain calls are made by the host module, the others by the Python form."""
import pytest
import torch

from heliopause_b200 import kernels as hk
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


class _Watched:
    """The host module, with what its functions answered."""

    def __init__(self, module):
        self.module, self.answers = module, []

    def __getattr__(self, name):
        def call(*args):
            got = getattr(self.module, name)(*args)
            self.answers.append(got is not NotImplemented)
            return got
        return call


@pytest.fixture
def watched(monkeypatch):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    hk.init_device(0)
    w = _Watched(hk._load_host())
    monkeypatch.setattr(hk, "_host", w)
    return w


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_which_calls_the_host_module_makes(watched, dtype):
    b = ref.Batch([40, 1, 0, 7], [340, 9, 3, 7], 2, 128, 16, dtype, spare_rows=2)
    x = torch.randn((b.rows, 12, 128), device="cuda", generator=b.gen)
    y = x.to(dtype)
    q, k, v = y[:, :8], y[:, 8:10], y[:, 10:]
    inv = torch.rand(32, device="cuda", dtype=torch.float64, generator=b.gen)
    norm = torch.rand(128, device="cuda", generator=b.gen)
    batch = (b.table, b.query_starts, b.kv_lens)
    key, value = b.key.clone(), b.value.clone()
    logits = torch.randn((3, 7001), device="cuda", generator=b.gen)
    i32 = lambda z: torch.tensor(z, dtype=torch.int32, device="cuda")  # noqa: E731
    ones = torch.ones(3, device="cuda")
    lists = dict(history=i32([5, 6, 6, 9]), history_starts=i32([0, 3, 3, 4]), prompt_lens=i32([1, 0, 0]), repetition=ones,
                 frequency=ones, presence=ones, bias_ids=i32([7, 8]), bias_values=ones[:2], bias_starts=i32([0, 1, 1, 2]),
                 allowed=torch.full((3, 219), -1, dtype=torch.int32, device="cuda"))

    def append(a=x, **kw):
        hk.paged_kv_append(a[:, 8:10], a[:, 10:], key, value, *batch, **kw)

    def paged(a=q, table=b.table, **kw):
        hk.paged_attention(a, b.key, b.value, table, b.query_starts, b.kv_lens, **{"max_query_len": 40, "scale": 0.1, **kw})

    def prompt(a=q, **kw):
        hk.prompt_attention(a, k, v, b.query_starts, **{"max_query_len": 40, "scale": 0.1, **kw})

    def by_the_module(call, *args, **kw):
        watched.answers.clear()
        call(*args, **kw)
        assert len(watched.answers) == 1
        return watched.answers[0]

    for call, args, kw in [
        (append, (), {}), (append, (y,), {}),
        (append, (), dict(q=x[:, :8], inv_freq=inv, q_norm=norm, k_norm=norm, norm_v=True, eps=1e-5)),
        (append, (), dict(q=x[:, :8], q_out=torch.empty((b.rows, 8, 128), dtype=dtype, device="cuda"))),
        (paged, (), {}), (paged, (), dict(window=7, scale=1)), (paged, (), dict(out_dtype=torch.float32)),
        (paged, (), dict(out=torch.empty_like(q, memory_format=torch.contiguous_format), max_query_len=1)),
        (prompt, (), {}), (prompt, (), dict(window=7, scale=1, max_query_len=1)), (prompt, (), dict(out_dtype=torch.float32)),
        (prompt, (), dict(out=torch.empty_like(q, memory_format=torch.contiguous_format))),
        (hk.logits_topk, (logits, 17), {}), (hk.logits_topk, (logits, 64), lists), (hk.logits_topk, (logits[:, 1:6001], 1), {}),
    ]:
        assert by_the_module(call, *args, **kw), (call.__name__, kw)
    odd = torch.empty(b.rows * 8 * 128 + 1, dtype=dtype, device="cuda")[1:].view(b.rows, 8, 128).copy_(q)
    for call, args, kw in [  # rows off 16 bytes, or not one behind the other: copied first
        (append, (x.transpose(1, 2).contiguous().transpose(1, 2),), {}), (paged, (odd,), {}), (prompt, (odd,), {}),
        (hk.logits_topk, (logits[:, ::2], 3), {}),
    ]:
        assert not by_the_module(call, *args, **kw), (call.__name__, kw)
    for call, args, kw in [
        (paged, (), dict(table=b.table.long())), (paged, (), dict(window=-1)), (prompt, (q[:5],), {}), (append, (), dict(eps=-1.0)),
        (hk.logits_topk, (logits, 65), {}), (hk.logits_topk, (logits, 3), dict(history=lists["history"])),
    ]:
        watched.answers.clear()
        with pytest.raises(hk.CudaKernelError):
            call(*args, **kw)
        assert watched.answers == [False]
