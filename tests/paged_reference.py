"""Plain 64-bit forms of the paged-cache operators, and the error their
16-bit results may have."""
import numpy as np
import torch


def rotate(x, pos, inv_freq):
    """NeoX rotation of [rows][heads][dim] (f64) by pos * inv_freq."""
    half = inv_freq.numel()
    ang = pos.double()[:, None, None] * inv_freq
    c, s = ang.cos(), ang.sin()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def rms(x, w, eps):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if w is None else y * w.double()


def positions(starts, lens, rows, device):
    """(sequence, position) of every packed row; -1 for rows of no sequence."""
    seq = torch.full((rows,), -1, dtype=torch.long)
    pos = torch.full((rows,), -1, dtype=torch.long)
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        seq[a:b] = s
        pos[a:b] = torch.arange(n - (b - a), n)
    return seq.to(device), pos.to(device)


def attention(q, k_of, v_of, starts, lens, scale, window):
    """f64 output, log-sum-exp, and per element the softmax-weighted |v| and
    the largest sum |q||k| * scale of its row's scores (for the tolerance).
    k_of(s), v_of(s): [len][kv_heads][dim] of sequence s."""
    rows, heads, dim = q.shape
    out = torch.zeros((rows, heads, dim), dtype=torch.float64, device=q.device)
    lse = torch.full((rows, heads), -torch.inf, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    smax = torch.zeros((rows, heads), dtype=torch.float64, device=q.device)
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        if a == b or n == 0:
            continue
        k, v = k_of(s).double(), v_of(s).double()
        group = heads // k.shape[1]
        pos = torch.arange(n - (b - a), n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)
        see = j <= pos
        if window:
            see &= j > pos - window
        for h in range(heads):
            qh, kh, vh = q[a:b, h].double(), k[:, h // group], v[:, h // group]
            w = torch.where(see, qh @ kh.T * scale, -torch.inf)
            m = w.amax(-1, keepdim=True)
            p = torch.where(see, torch.exp(w - torch.where(m > -torch.inf, m, 0.0)), 0.0)
            l = p.sum(-1, keepdim=True)
            # a key that is not seen adds nothing, whatever its value holds
            o = torch.stack([(p[i][see[i]][:, None] * vh[see[i]]).sum(0) for i in range(b - a)]) \
                if not torch.isfinite(vh).all() else p @ vh
            out[a:b, h] = torch.where(l > 0, o / l, 0.0)
            mag[a:b, h] = torch.where(l > 0, (p @ torch.nan_to_num(vh).abs()) / l, 0.0)
            lse[a:b, h] = (torch.log(l) + m)[:, 0]
            t = torch.where(see, qh.abs() @ kh.abs().T * abs(scale), 0.0)
            smax[a:b, h] = torch.nan_to_num(t).amax(-1)
    return out, lse, mag, smax


def attention_tolerance(dtype, out_dtype, mag, smax, dim, keys):
    """Half a step for each rounding: of the probabilities (to the cache's
    type, a relative u each, so u times the weighted |v|) and of the output;
    the scores are f32 sums of `dim` products (dim steps of 2^-23 of the sum of
    their sizes, as an error of the exponent on both sides of the division);
    the output is an f32 sum over the keys and the joined parts; exp2 is good to
    2^-21."""
    u = torch.finfo(dtype).eps / 2
    uo = torch.finfo(out_dtype).eps / 2
    rel = u + uo + 2 * (dim * 2.0 ** -23 * smax[..., None] + 2.0 ** -21) + (keys + 64) * 2.0 ** -23
    return rel * mag + torch.finfo(out_dtype).smallest_normal * uo * 2


class Batch:
    """Ragged sequences over a shuffled paged cache; slots of no token, and
    pages of no sequence, hold NaN."""

    def __init__(self, new, lens, kv_heads, dim, page, dtype, seed=0, spare_rows=0, device="cuda", spare_width=2):
        g = torch.Generator(device=device).manual_seed(seed)
        self.new, self.lens, self.page = list(new), list(lens), page
        self.starts = [int(x) for x in np.concatenate([[0], np.cumsum(new)])]
        self.rows = self.starts[-1] + spare_rows
        per = [-(-n // page) for n in lens]
        pages = sum(per) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max([1] + per) + spare_width
        table = torch.full((len(lens), width), -7, dtype=torch.int32)  # entries of no token are never followed
        self.key = torch.full((pages, page, kv_heads, dim), torch.nan, dtype=dtype, device=device)
        self.value = torch.full_like(self.key, torch.nan)
        self.slots = []
        for s, n in enumerate(lens):
            own, order = order[:per[s]], order[per[s]:]
            table[s, :per[s]] = torch.tensor(own, dtype=torch.int32)
            j = torch.arange(n)
            slot = torch.tensor(own, dtype=torch.long)[j // page] * page + j % page if n else j
            slot = slot.to(device)
            self.slots.append(slot)
            for c in (self.key, self.value):
                c.view(-1, kv_heads, dim)[slot] = torch.randn((n, kv_heads, dim), device=device, generator=g).to(dtype)
        self.table = table.to(device)
        self.query_starts = torch.tensor(self.starts, dtype=torch.int32, device=device)
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.gen = g

    def k_of(self, s):
        return self.key.view(-1, *self.key.shape[2:])[self.slots[s]]

    def v_of(self, s):
        return self.value.view(-1, *self.value.shape[2:])[self.slots[s]]
