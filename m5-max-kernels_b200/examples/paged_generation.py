"""Decoding with a quantized attention layer over a paged cache.

    python m5-max-kernels_b200/examples/paged_generation.py

One attention layer of 4096 channels (32 query heads, 8 key/value heads of 128)
the way a serving loop runs it: RMSNorm and INT8 codes (`rms_quantize`), one
W8A8 product for queries, keys and values (`gemm`), rotation and the new keys
and values into the cache's pages (`paged_append`), attention of the new tokens
over it (`paged_attention`), and the quantized output projection (`linear`).
Sequences of different lengths enter chunk by chunk, mixed with others that
already decode, get pages as they grow and give them back.  At the end the
chunked outputs are compared with those of every sequence as one whole prompt.
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import m5kernels_b200 as m

HEAD_DIM = 128


class PagedCache:
    """Pages of keys and values, and which sequence has which (kept on the host)."""

    def __init__(self, pages, page, kv_heads, device, dtype=torch.bfloat16):
        shape = (pages, kv_heads, page, HEAD_DIM)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.page, self.device = page, device
        self.free = list(range(pages))
        self.tables: dict = {}
        self.lengths: dict = {}

    def extend(self, seq, tokens):
        """Room for `tokens` more tokens of sequence `seq`."""
        table = self.tables.setdefault(seq, [])
        length = self.lengths.get(seq, 0) + tokens
        while len(table) * self.page < length:
            if not self.free:
                raise MemoryError("the cache has no free page")
            table.append(self.free.pop())
        self.lengths[seq] = length

    def release(self, seq):
        self.free += self.tables.pop(seq)
        del self.lengths[seq]

    def batch(self, seqs, tokens):
        """page_table, query_start, seq_lens of a batch, one copy to the device each."""
        width = max(len(self.tables[s]) for s in seqs)
        table = [self.tables[s] + [-1] * (width - len(self.tables[s])) for s in seqs]
        starts = [0]
        for n in tokens:
            starts.append(starts[-1] + n)
        put = lambda x: torch.tensor(x, dtype=torch.int32).to(self.device, non_blocking=True)
        return put(table), put(starts), put([self.lengths[s] for s in seqs])


class AttentionLayer:
    """x + out(attention(rope(qkv(rms(x))))) with INT8 weights and activations."""

    def __init__(self, width, q_heads, kv_heads, positions, device, seed=0, block=128):
        g = torch.Generator().manual_seed(seed)
        heads = q_heads + 2 * kv_heads
        w_qkv = torch.randn(heads * HEAD_DIM, width, generator=g) * width**-0.5
        w_out = torch.randn(width, q_heads * HEAD_DIM, generator=g) * (q_heads * HEAD_DIM) ** -0.5
        self.q_heads, self.kv_heads, self.block = q_heads, kv_heads, block
        self.gamma = torch.ones(width, device=device)
        self.signs = (torch.randint(0, 2, (width,), generator=g) * 2 - 1).to(torch.int8).to(device)
        self.w_qkv, self.s_qkv = m.hadamard_quantize(w_qkv.to(torch.bfloat16).to(device), block,
                                                     self.signs, "int8")
        self.w_out, self.s_out = m.quantize(w_out.to(torch.bfloat16).to(device), "int8")
        self.cos, self.sin = m.rope_tables(positions, HEAD_DIM // 2, device=device)

    def __call__(self, x, cache, page_table, query_start, seq_lens, max_query_len):
        codes, scales = m.rms_quantize(x, self.gamma, self.signs, self.block)
        rows = m.gemm(codes, self.w_qkv, "int8", a_scales=scales, b_scales=self.s_qkv,
                      output_dtype=torch.bfloat16).view(x.shape[0], -1, HEAD_DIM)
        q, k, v = rows.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)
        q = m.paged_append(k, v, cache.k, cache.v, page_table, query_start, seq_lens,
                           cos=self.cos, sin=self.sin, q=q)
        o = m.paged_attention(q, cache.k, cache.v, page_table, query_start, seq_lens,
                              max_query_len=max_query_len)
        return x + m.linear(o.view(x.shape[0], -1), self.w_out, self.s_out)


def serve(layer, cache, inputs, chunk):
    """All rows of `inputs` (one [tokens, width] tensor a sequence) through the layer.

    A new sequence joins at every step; each brings `chunk` tokens a step while
    it has that many left, then one at a time, as if it were generating.
    """
    done, outs, step = [0] * len(inputs), [[] for _ in inputs], 0
    while any(d < len(x) for d, x in zip(done, inputs)):
        step += 1
        seqs = [s for s in range(min(step, len(inputs))) if done[s] < len(inputs[s])]
        if not seqs:
            continue
        tokens = [chunk if len(inputs[s]) - done[s] > chunk else 1 for s in seqs]
        x = torch.cat([inputs[s][done[s]:done[s] + n] for s, n in zip(seqs, tokens)])
        for s, n in zip(seqs, tokens):
            cache.extend(s, n)
        y = layer(x, cache, *cache.batch(seqs, tokens), max(tokens))
        at = 0
        for s, n in zip(seqs, tokens):
            outs[s].append(y[at:at + n])
            done[s] += n
            at += n
            if done[s] == len(inputs[s]):
                cache.release(s)
    return [torch.cat(o) for o in outs], step


def main(width=4096, q_heads=32, kv_heads=8, lengths=(700, 37, 264, 1, 513), chunk=96, page=16,
         device="cuda"):
    device = torch.device(device, torch.cuda.current_device())
    g = torch.Generator().manual_seed(1)
    inputs = [torch.randn(n, width, generator=g).to(torch.bfloat16).to(device) for n in lengths]
    layer = AttentionLayer(width, q_heads, kv_heads, max(lengths), device)
    pages = sum(-(-n // page) for n in lengths)
    served, steps = serve(layer, PagedCache(pages, page, kv_heads, device), inputs, chunk)
    whole = PagedCache(pages, page, kv_heads, device)
    worst = 0.0
    for s, (x, y) in enumerate(zip(inputs, served)):
        whole.extend(s, len(x))
        ref = layer(x, whole, *whole.batch([s], [len(x)]), len(x))
        # the layer's own contribution, apart from x: codes may differ by one where
        # the attention kernels round differently
        a, b = (y - x).double(), (ref - x).double()
        worst = max(worst, float((a - b).norm() / b.norm()))
    print(f"{len(inputs)} sequences, {sum(lengths)} tokens in {steps} steps; "
          f"chunked against whole prompts: relative L2 {worst:.2e}")
    return worst


if __name__ == "__main__":
    sys.exit(0 if main() < 2e-2 else 1)
