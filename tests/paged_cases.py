"""Paged batches for the tests, and the 64-bit oracle of the two operators."""

import math
import random

import torch

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


class Batch:
    """A ragged batch with its cache, on the CPU.

    Slots that hold no token are NaN, page numbers behind a sequence's last
    page are -1, pages are in random order.
    """

    def __init__(self, new, ctx, *, q_heads, kv_heads, dim, page, dtype, seed=0, fill=math.nan,
                 pad_rows=0, lead_rows=0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.page, self.dtype = list(new), page, dtype
        self.seq = [n + c for n, c in zip(new, ctx)]  # ctx < 0: fewer keys than tokens
        starts = [lead_rows]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts, self.rows = starts, starts[-1] + pad_rows
        pages = [-(-max(s, 0) // page) for s in self.seq]
        self.num_pages, width = sum(pages) + 2, max(max(pages), 1)
        order = list(range(self.num_pages))
        random.Random(seed).shuffle(order)
        self.table = torch.full((len(new), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        shape = (self.num_pages, kv_heads, page, dim)
        self.k_cache = torch.full(shape, fill, dtype=dtype)
        self.v_cache = torch.full(shape, fill, dtype=dtype)
        self.k, self.v = [], []
        for b, s in enumerate(self.seq):
            k = torch.randn(max(s, 0), kv_heads, dim, generator=g).to(dtype)
            v = torch.randn(max(s, 0), kv_heads, dim, generator=g).to(dtype)
            self.k.append(k)
            self.v.append(v)
            for p in range(max(s, 0)):
                self.k_cache[self.table[b, p // page], :, p % page] = k[p]
                self.v_cache[self.table[b, p // page], :, p % page] = v[p]
        self.q = (1.5 * torch.randn(self.rows, q_heads, dim, generator=g)).to(dtype)
        self.query_start = torch.tensor(starts, dtype=torch.int32)
        self.seq_lens = torch.tensor(self.seq, dtype=torch.int32)

    def on(self, dev):
        return [t.to(dev) for t in (self.k_cache, self.v_cache, self.table, self.query_start,
                                    self.seq_lens)]


def attend_oracle(batch, *, scale=None, softcap=None, slopes=None, window=None, prefix=None):
    """(out, lse, spread) in 64 bits; spread = sum of p |v| per output channel."""
    rows, heads, dim = batch.q.shape
    group = heads // batch.k_cache.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    for b, (n, length) in enumerate(zip(batch.new, batch.seq)):
        if n == 0 or length <= 0:
            continue
        pos = torch.arange(length - n, length)[:, None]
        key = torch.arange(length)[None, :]
        seen = key <= pos
        if window is not None:
            seen &= pos - key < window
        if prefix is not None:
            seen |= key < prefix[b]
        lo = batch.starts[b]
        for h in range(heads):
            k, v = batch.k[b][:, h // group].double(), batch.v[b][:, h // group].double()
            x = batch.q[lo:lo + n, h].double() @ k.T * scale
            if softcap is not None:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * (pos - key).abs()
            x = x.masked_fill(~seen, -math.inf)
            z = torch.logsumexp(x, 1)
            p = torch.where(seen, torch.exp(x - torch.where(z.isinf(), 0.0, z)[:, None]), 0.0)
            out[lo:lo + n, h], spread[lo:lo + n, h] = p @ v, p @ v.abs()
            lse[lo:lo + n, h] = z
    return out, lse, spread


def check_attention(got, lse, want, want_lse, spread, dtype):
    """|error| <= u |o| + (u + e) sum p |v|, u the type's unit roundoff.

    The first term is the output's rounding, the second that of the
    probabilities to the type of V and e for the scores and the exponentials:
    2^-11 for the 16-bit types, 2^-16 for fp32.  The logarithm has no rounded
    probabilities: e and 2^-20 of itself.
    """
    u, e = UNIT[dtype], 2.0**-16 if dtype == torch.float32 else 2.0**-11
    assert torch.isfinite(got).all()
    excess = (got.double().cpu() - want).abs() - (u * want.abs() + (u + e) * spread + 1e-30)
    assert excess.max().item() <= 0, excess.max().item()
    if lse is not None:
        lse = lse.double().cpu()
        empty = want_lse.isinf()
        assert torch.equal(lse.isinf(), empty) and (lse[empty] < 0).all()
        off = (lse - want_lse)[~empty].abs() - (e + 2.0**-20 * want_lse[~empty].abs())
        assert off.numel() == 0 or off.max().item() <= 0, off.max().item()


def rotate_oracle(x, cos, sin, layout):
    """x [n, heads, dim] turned by cos, sin [n, R], in 64 bits."""
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    r = cos.shape[-1]
    y = x.clone()
    i, j = ((slice(0, r), slice(r, 2 * r)) if layout == "half"
            else (slice(0, 2 * r, 2), slice(1, 2 * r, 2)))
    y[..., i] = x[..., i] * cos - x[..., j] * sin
    y[..., j] = x[..., j] * cos + x[..., i] * sin
    return y
