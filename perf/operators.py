"""The serving operators' cases: plain forms, the framework's calls, and 64-bit values.

Four operators of a batch that is served from a paged key-value cache:

append    new tokens' keys and values into the pages (per-head RMS norms and
          the position rotation on the way), the rotated queries out;
paged     causal attention of each sequence's newest tokens over its pages
          (one token, a few drafts, or a chunk of a prompt);
prompt    causal attention over whole prompts, packed one behind the other;
logits    penalties, biases and a grammar mask on logits, and the k best.

Sequence s owns the rows query_starts[s] .. query_starts[s + 1] of the packed
tensors; kv_lens[s] is its length with those rows counted in; token j of it
lies in page page_table[s][j / page_size].
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 64 running chats: the framework's decoder (8 query and 2 KV heads of 256, QK and V norms)
        {"name": "append-decode", "op": "append", "seqs": 64, "new_lo": 1, "new_hi": 1, "past": 900, "heads": 8, "kv_heads": 2,
         "dim": 256, "rot": 256, "page": 16, "dtype": "f16", "norm": True},
        # five prompts entering the cache at once, generic heads without norms, half of each head rotated
        {"name": "append-prompts", "op": "append", "seqs": 5, "new_lo": 311, "new_hi": 1600, "past": 300, "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 64, "page": 64, "dtype": "bf16", "norm": False},
        # one chat at the framework's full context: the latency of a single token
        {"name": "paged-one", "op": "paged", "seqs": 1, "new_lo": 1, "new_hi": 1, "kv_lo": 4096, "kv_hi": 4096, "heads": 8,
         "kv_heads": 2, "dim": 256, "page": 16, "dtype": "f16", "window": 0},
        # 64 chats of every length up to that context
        {"name": "paged-ragged", "op": "paged", "seqs": 64, "new_lo": 1, "new_hi": 1, "kv_lo": 1, "kv_hi": 4096, "heads": 8,
         "kv_heads": 2, "dim": 256, "page": 16, "dtype": "bf16", "window": 0},
        # the verify step: a pending token and four drafts of each of 16 chats
        {"name": "paged-verify", "op": "paged", "seqs": 16, "new_lo": 5, "new_hi": 5, "kv_lo": 1000, "kv_hi": 4096, "heads": 8,
         "kv_heads": 2, "dim": 256, "page": 64, "dtype": "f16", "window": 0},
        # long documents being answered: generic heads
        {"name": "paged-long", "op": "paged", "seqs": 32, "new_lo": 1, "new_hi": 1, "kv_lo": 8192, "kv_hi": 32768, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "window": 0},
        # chunks of four long prompts against what the cache already holds
        {"name": "paged-chunk", "op": "paged", "seqs": 4, "new_lo": 384, "new_hi": 512, "kv_lo": 2000, "kv_hi": 8192, "heads": 8,
         "kv_heads": 2, "dim": 256, "page": 64, "dtype": "bf16", "window": 0},
        # a short question: the framework's heads
        {"name": "prompt-short", "op": "prompt", "seqs": 1, "new_lo": 333, "new_hi": 333, "heads": 8, "kv_heads": 2, "dim": 256,
         "dtype": "f16", "window": 0},
        # twelve prompts of very different lengths in one pass
        {"name": "prompt-packed", "op": "prompt", "seqs": 12, "new_lo": 1, "new_hi": 2048, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "f16", "window": 0},
        # one long prompt
        {"name": "prompt-long", "op": "prompt", "seqs": 1, "new_lo": 8192, "new_hi": 8192, "heads": 8, "kv_heads": 2, "dim": 256,
         "dtype": "bf16", "window": 0},
        # one chat's next token over the framework's vocabulary
        {"name": "logits-one", "op": "logits", "rows": 1, "vocab": 262144, "k": 64, "hist_lo": 700, "hist_hi": 700, "bias": 0,
         "mask": False},
        # 64 chats with histories, biases and a grammar each
        {"name": "logits-batch", "op": "logits", "rows": 64, "vocab": 262144, "k": 40, "hist_lo": 1, "hist_hi": 4096, "bias": 50,
         "mask": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "paged", "paged", "prompt", "prompt", "logits"])
    dtype = rng.choice(["f16", "bf16"])
    dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 7, 8] if kv_heads < 8 else [1, 2, 4])
    page = rng.choice([16, 32, 64, 128])
    window = rng.choice([0, 0, 0, _log_int(rng, 1, 4000)])
    if op == "append":
        new = _log_int(rng, 1, 1024)
        seqs = _log_int(rng, 1, max(1, min(128, 8192 // new)))
        return {"op": op, "seqs": seqs, "new_lo": max(1, new // 3), "new_hi": new, "past": _log_int(rng, 1, 1500), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rot": dim // rng.choice([1, 1, 2]), "page": page, "dtype": dtype,
                "norm": rng.random() < 0.5}
    if op == "paged":
        new = rng.choice([1, 1, 1, 2, 5, 8, _log_int(rng, 9, 600)])
        hi = _log_int(rng, max(16, new), 16384)
        most = max(1, 4_000_000 * 128 // (hi * kv_heads * dim))
        if new > 8:
            most = max(1, min(most, 480_000_000 // (hi * new * heads), 60_000_000_000 // (hi * new * heads * dim)))
        return {"op": op, "seqs": _log_int(rng, 1, min(128, most)), "new_lo": new, "new_hi": new, "kv_lo": max(new, hi // rng.choice([1, 3, 20])),
                "kv_hi": hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "window": window}
    if op == "prompt":
        hi = min(_log_int(rng, 1, 8192), math.isqrt(120_000_000_000 // (heads * dim)))
        most = max(1, min(1_280_000_000 // (hi * hi * heads), 120_000_000_000 // (hi * hi * heads * dim)))
        return {"op": op, "seqs": _log_int(rng, 1, min(24, most)), "new_lo": max(1, hi // rng.choice([1, 4, 30])), "new_hi": hi,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "window": window}
    vocab = _log_int(rng, 2000, 300000)
    hist = _log_int(rng, 1, 5000)
    return {"op": op, "rows": _log_int(rng, 1, 100), "vocab": vocab, "k": rng.randint(1, 64), "hist_lo": max(1, hist // 5), "hist_hi": hist,
            "bias": rng.choice([0, _log_int(rng, 1, 300)]), "mask": rng.random() < 0.5}


# ---- inputs --------------------------------------------------------------------------------

def _spread(case, lo, hi, n):
    """n lengths from lo to hi, both among them where there are two, the rest at places fixed by the case."""
    if n == 1 or lo == hi:
        return [hi] * n
    mid = [lo + (hi - lo) * ((i * 0.6180339887498949) % 1.0) for i in range(1, n - 1)]
    return [hi] + [int(x) for x in mid] + [lo]


def _lengths(case):
    """(new tokens, length with them) of every sequence."""
    n = case["seqs"]
    new = _spread(case, case["new_lo"], case["new_hi"], n)
    if case["op"] == "append":
        return new, [t + (case["past"] * (i + 1)) // n for i, t in enumerate(new)]
    if case["op"] == "paged":
        return new, [max(t, x) for t, x in zip(new, reversed(_spread(case, case["kv_lo"], case["kv_hi"], n)))]
    return new, list(new)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    def whole(hi, *shape):
        return torch.randint(0, hi, shape, device="cuda", generator=gen, dtype=torch.int32)

    def counted(xs):
        return torch.tensor([sum(xs[:i]) for i in range(len(xs) + 1)], dtype=torch.int32, device="cuda")

    st = {"case": dict(case), "op": case["op"]}
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        st["logits"] = randn(rows, vocab) * 3
        hist = _spread(case, case["hist_lo"], case["hist_hi"], rows)
        starts = counted(hist)
        # a history repeats itself: tokens come from a tenth of their number of distinct ids
        pool = whole(vocab, max(2, max(hist) // 2))
        st["history"] = pool[whole(pool.numel(), sum(hist)).long()]
        st["history_starts"] = starts
        st["prompt_lens"] = torch.tensor([h // 3 for h in hist], dtype=torch.int32, device="cuda")
        st["repetition"] = 1.0 + 0.5 * torch.rand(rows, device="cuda", generator=gen)
        st["frequency"] = 0.5 * torch.rand(rows, device="cuda", generator=gen)
        st["presence"] = torch.rand(rows, device="cuda", generator=gen) - 0.25
        if case["bias"]:
            n = case["bias"] * rows
            st["bias_starts"] = counted([case["bias"]] * rows)
            st["bias_ids"] = whole(vocab, n)
            st["bias_values"] = randn(n) * 5
        if case["mask"]:
            # a grammar's allowed tokens, one bit a token
            words = torch.randint(-2**31, 2**31, (2, rows, (vocab + 31) // 32), device="cuda", generator=gen, dtype=torch.int64)
            st["allowed"] = (words[0] & words[1]).to(torch.int32)
        return st

    dt = DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    new, lens = _lengths(case)
    total = sum(new)
    st["query_starts"] = counted(new)
    st["max_len"] = max(new)
    st["scale"] = 1.0 / math.sqrt(dim)
    if case["op"] == "prompt":
        # the projections' output, cut into its three parts: strided views
        qkv = randn(total, heads + 2 * kv_heads, dim)
        qkv[:, :heads] *= 1.5
        qkv = qkv.to(dt)
        st["q"], st["k"], st["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        return st
    page = case["page"]
    per = [(x + page - 1) // page for x in lens]
    pages = sum(per) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((case["seqs"], max(per)), dtype=torch.int32)
    at = 0
    host = order.cpu()
    for s, n in enumerate(per):
        table[s, :n] = host[at:at + n]
        at += n
    st["page_table"] = table.cuda()
    st["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["key_cache"] = randn(pages, page, kv_heads, dim).to(dt)
    st["value_cache"] = randn(pages, page, kv_heads, dim).to(dt)
    if case["op"] == "paged":
        st["q"] = (randn(total, heads, dim) * 1.5).to(dt)
        return st
    qkv = randn(total, heads + 2 * kv_heads, dim) * 2
    st["q"], st["k"], st["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    half = case["rot"] // 2
    st["inv_freq"] = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    if case["norm"]:
        st["q_norm"] = 1 + 0.1 * randn(dim)
        st["k_norm"] = 1 + 0.1 * randn(dim)
    return st


# ---- one pass ------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if own:
        from heliopause_b200 import kernels as hk

        if st["op"] == "append":
            q = hk.paged_kv_append(st["k"], st["v"], st["key_cache"], st["value_cache"], st["page_table"], st["query_starts"],
                                   st["kv_lens"], q=st["q"], inv_freq=st["inv_freq"], q_norm=st.get("q_norm"),
                                   k_norm=st.get("k_norm"), norm_v=case["norm"], eps=1e-6)
            return {"q": q, "key_cache": st["key_cache"], "value_cache": st["value_cache"]}
        if st["op"] == "paged":
            return hk.paged_attention(st["q"], st["key_cache"], st["value_cache"], st["page_table"], st["query_starts"],
                                      st["kv_lens"], max_query_len=st["max_len"], scale=st["scale"], window=case["window"])
        if st["op"] == "prompt":
            return hk.prompt_attention(st["q"], st["k"], st["v"], st["query_starts"], max_query_len=st["max_len"],
                                       scale=st["scale"], window=case["window"])
        ids, vals = hk.logits_topk(st["logits"], case["k"], history=st["history"], history_starts=st["history_starts"],
                                   prompt_lens=st["prompt_lens"], repetition=st["repetition"], frequency=st["frequency"],
                                   presence=st["presence"], bias_ids=st.get("bias_ids"), bias_values=st.get("bias_values"),
                                   bias_starts=st.get("bias_starts"), allowed=st.get("allowed"))
        return {"ids": ids, "vals": vals}
    if st["op"] == "append":
        return _plain_append(st)
    if st["op"] == "logits":
        return _plain_logits(st)
    return _plain_attention(st)


def _rows(st, total):
    """(sequence, position) of every packed row."""
    starts = st["query_starts"].long()
    row = torch.arange(total, device=starts.device)
    seq = torch.searchsorted(starts, row, right=True) - 1
    new = starts[1:] - starts[:-1]
    return seq, st["kv_lens"].long()[seq] - new[seq] + row - starts[seq]


def _rms(x, w):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return y if w is None else y * w


def _rotate(x, cos, sin):
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _plain_append(st):
    norm, page = st["case"]["norm"], st["case"]["page"]
    q, k, v = st["q"], st["k"], st["v"]
    seq, pos = _rows(st, k.shape[0])
    if norm:
        q, k, v = _rms(q, st["q_norm"]), _rms(k, st["k_norm"]), _rms(v, None)
    angle = pos.double()[:, None, None] * st["inv_freq"]  # far positions: 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    at = st["page_table"].long()[seq, pos // page]
    dt = st["key_cache"].dtype
    st["key_cache"][at, pos % page] = _rotate(k, cos, sin).to(dt)
    st["value_cache"][at, pos % page] = v.to(dt)
    return {"q": _rotate(q, cos, sin).to(dt), "key_cache": st["key_cache"], "value_cache": st["value_cache"]}


def _plain_attention(st):
    """Every sequence padded to the longest: [sequence][KV head][group * query][key]."""
    q, starts, window = st["q"], st["query_starts"].long(), st["case"]["window"]
    total, heads, dim = q.shape
    new = starts[1:] - starts[:-1]
    seqs, most = new.numel(), st["max_len"]
    dev = q.device
    row = starts[:-1, None] + torch.arange(most, device=dev)
    row = torch.where(torch.arange(most, device=dev) < new[:, None], row, 0)
    if st["op"] == "paged":
        lens, page = st["kv_lens"].long(), st["case"]["page"]
        j = torch.arange(st["page_table"].shape[1] * page, device=dev)
        at = st["page_table"].long()[:, j // page]
        k, v = st["key_cache"][at, j % page].float(), st["value_cache"][at, j % page].float()
    else:
        lens, j = new, torch.arange(most, device=dev)
        k, v = st["k"][row].float(), st["v"][row].float()
    kv_heads = k.shape[2]
    group = heads // kv_heads
    qs = q[row].float() * st["scale"]  # [S][L][H][D]
    qs = qs.view(seqs, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * most, dim)
    k, v = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)
    s = torch.matmul(qs, k).view(seqs, kv_heads, group, most, j.numel())
    pos = (lens - new)[:, None] + torch.arange(most, device=dev)
    see = (j <= pos[..., None]) & (j < lens[:, None, None])
    if window:
        see &= j > pos[..., None] - window
    s.masked_fill_(~see[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True).clamp_min(-1e30)
    s.exp_()
    s /= s.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(s.view(seqs, kv_heads, group * most, j.numel()), v)
    o = o.view(seqs, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    return o[torch.arange(most, device=dev) < new[:, None]].to(q.dtype)


def _counts(st, rows, vocab):
    """(seen anywhere, times in the output) of every token of every row."""
    hist, starts = st["history"].long(), st["history_starts"].long()
    at = torch.arange(hist.numel(), device=hist.device)
    row = torch.searchsorted(starts, at, right=True) - 1
    out = at - starts[row] >= st["prompt_lens"].long()[row]
    flat = row * vocab + hist
    seen = torch.zeros(rows * vocab, dtype=torch.bool, device=hist.device)
    seen[flat] = True
    times = torch.zeros(rows * vocab, dtype=torch.int32, device=hist.device).scatter_add_(0, flat, out.int())
    return seen.view(rows, vocab), times.view(rows, vocab)


def _plain_logits(st):
    """The values in 64 bits, rounded once: what lies next to another is ranked by it."""
    x, k = st["logits"].double(), st["case"]["k"]
    rows, vocab = x.shape
    seen, times = _counts(st, rows, vocab)
    r = st["repetition"].double()[:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"].double()[:, None] * times - st["presence"].double()[:, None] * (times > 0)
    if "bias_ids" in st:
        row = torch.searchsorted(st["bias_starts"].long(), torch.arange(st["bias_ids"].numel(), device=x.device), right=True) - 1
        x.index_put_((row, st["bias_ids"].long()), st["bias_values"].double(), accumulate=True)
    if "allowed" in st:
        bit = (st["allowed"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bit.view(rows, -1)[:, :vocab] == 0, -math.inf)
    vals, ids = x.float().sort(dim=-1, descending=True, stable=True)
    vals, ids = vals[:, :k].contiguous(), ids[:, :k].int()
    return {"ids": torch.where(vals > -math.inf, ids, -1), "vals": vals}


# ---- the same from the definition, in 64 bits -------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(st)
    if case["op"] == "logits":
        return _exact_logits(st)
    return _exact_attention(st)


def _exact_append(st):
    case = st["case"]
    new, lens = _lengths(case)
    kc, vc = st["key_cache"].double(), st["value_cache"].double()
    qo = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    half = case["rot"] // 2
    at = 0
    for s, (t, n) in enumerate(zip(new, lens)):
        q, k, v = (st[x][at:at + t].double() for x in "qkv")
        if case["norm"]:
            q = q / ((q ** 2).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt() * st["q_norm"].double()
            k = k / ((k ** 2).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt() * st["k_norm"].double()
            v = v / ((v ** 2).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt()
        pos = torch.arange(n - t, n, device="cuda")
        turn = torch.polar(torch.ones(t, 1, half, dtype=torch.float64, device="cuda"),
                           pos[:, None, None].double() * st["inv_freq"])
        for x in (q, k):
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            x[..., :half], x[..., half:2 * half] = z.real, z.imag
        slot = st["page_table"][s].long()[pos // case["page"]] * case["page"] + pos % case["page"]
        kc.view(-1, *kc.shape[2:])[slot] = k
        vc.view(-1, *vc.shape[2:])[slot] = v
        qo[at:at + t] = q
        at += t
    return {"q": qo, "key_cache": kc, "value_cache": vc}


def _exact_attention(st):
    case = st["case"]
    new, lens = _lengths(case)
    if case["op"] == "prompt":
        lens = new
    heads, kv_heads = case["heads"], case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (t, n) in enumerate(zip(new, lens)):
        if case["op"] == "paged":
            j = torch.arange(n, device="cuda")
            slot = st["page_table"][s].long()[j // case["page"]] * case["page"] + j % case["page"]
            k = st["key_cache"].view(-1, kv_heads, case["dim"])[slot].double()
            v = st["value_cache"].view(-1, kv_heads, case["dim"])[slot].double()
        else:
            k, v = st["k"][at:at + t].double(), st["v"][at:at + t].double()
        for h in range(heads):
            g = h // (heads // kv_heads)
            for a in range(0, t, 2048):
                b = min(t, a + 2048)
                w = st["q"][at + a:at + b, h].double() @ k[:, g].T * st["scale"]
                far = torch.arange(n - t + a, n - t + b, device="cuda")[:, None] - torch.arange(n, device="cuda")
                hide = far < 0
                if case["window"]:
                    hide |= far >= case["window"]
                w[hide] = -math.inf
                out[at + a:at + b, h] = torch.softmax(w, -1) @ v[:, g]
        at += t
    return out


def _exact_logits(st):
    case = st["case"]
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    hist = st["history"].long().split((st["history_starts"][1:] - st["history_starts"][:-1]).tolist())
    ids, vals = [], []
    for r in range(rows):
        x = st["logits"][r].double()
        seen = torch.bincount(hist[r], minlength=vocab) > 0
        times = torch.bincount(hist[r][int(st["prompt_lens"][r]):], minlength=vocab)
        rep = st["repetition"][r].double()
        x[seen & (x > 0)] /= rep
        x[seen & (st["logits"][r] <= 0)] *= rep
        x -= times * st["frequency"][r].double() + (times > 0) * st["presence"][r].double()
        if "bias_ids" in st:
            n = case["bias"]
            x.index_add_(0, st["bias_ids"][r * n:(r + 1) * n].long(), st["bias_values"][r * n:(r + 1) * n].double())
        live = torch.ones(vocab, dtype=torch.bool, device="cuda")
        if "allowed" in st:
            i = torch.arange(vocab, device="cuda")
            live = (st["allowed"][r].long()[i // 32] >> (i % 32)) & 1 == 1
        at = live.nonzero().flatten()
        # ranked as the f32 values that are handed out, ties by id
        got, order = x[at].float().sort(descending=True, stable=True)
        n = min(k, at.numel())
        top = at[order[:n]]
        ids.append(torch.cat([top, torch.full((k - n,), -1, device="cuda")]).int())
        vals.append(torch.cat([x[top], torch.full((k - n,), -math.inf, dtype=torch.float64, device="cuda")]))
    return {"ids": torch.stack(ids), "vals": torch.stack(vals)}


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        hist = sum(_spread(case, case["hist_lo"], case["hist_hi"], rows))
        b = rows * (4 * vocab + 8 * case["k"] + 12) + 4 * hist + 8 * case["bias"] * rows + (rows * vocab // 8 if case["mask"] else 0)
        return {"bytes": b, "flops": rows * vocab + 4 * hist}
    new, lens = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    total = sum(new)
    if case["op"] == "append":
        return {"bytes": total * (heads + 2 * kv_heads) * dim * (4 + 2), "flops": total * (heads + kv_heads) * dim * (6 if case["norm"] else 3)}
    window = case["window"] or 1 << 60
    pairs = keys = 0
    for t, n in zip(new, lens):
        first = n - t  # position of the first new token
        # sum over positions p of min(p + 1, window)
        full = max(0, min(n, window) - first)
        pairs += full * (2 * first + full + 1) // 2 + (t - full) * min(window, n)
        keys += min(n, window + t - 1)
    return {"bytes": 2 * (2 * total * heads * dim + 2 * keys * kv_heads * dim), "flops": 4 * pairs * heads * dim}
