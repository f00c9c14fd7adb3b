"""The paged cache on the GPU: appending and attention against 64-bit oracles."""

import math

import pytest
import torch

from paged_cases import (UNIT, Batch, attend_oracle, check_attention, rotate_oracle)

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m
    from m5kernels_b200 import _lib

    yield m
    assert _lib.device_status() == 0  # no bounded wait gave up


def attend(ops, batch, *, hint=None, **kw):
    prefix = kw.pop("prefix", None)
    slopes = kw.pop("slopes", None)
    return ops.paged_attention(
        batch.q.to(DEV), *batch.on(DEV),
        max_query_len=max(batch.new) if hint is None else hint, return_lse=True,
        slopes=None if slopes is None else slopes.to(DEV),
        prefix_lens=None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=DEV),
        **kw)


def compare(ops, batch, **kw):
    want, want_lse, spread = attend_oracle(
        batch, **{k: v for k, v in kw.items() if k != "hint"})
    out, lse = attend(ops, batch, **kw)
    check_attention(out, lse, want, want_lse, spread, batch.dtype)
    return out


# new tokens and cached tokens per sequence: single tokens; drafts; chunks; whole prompts; mixtures
# with sequences without new tokens, of length zero, and with fewer keys than tokens
RAGGED = {
    "one": ([1], [0]),
    "short": ([1], [16]),
    "decode": ([1, 1, 1, 1], [0, 63, 64, 517]),
    "drafts": ([5, 3, 4], [100, 0, 259]),
    "chunk": ([70], [130]),
    "prompt": ([300, 129], [0, 0]),
    "mixed": ([1, 200, 0, 7, 1, 33], [300, 0, 50, 121, 0, 128]),
    "empty_rows": ([1, 40, 3, 1], [-1, -10, -3, 5]),
}


@pytest.mark.parametrize("ragged", RAGGED)
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype", [
    (8, 2, 128, 16, BF16), (4, 4, 64, 32, F16), (6, 2, 128, 64, F16), (8, 1, 64, 128, BF16),
    (7, 1, 128, 256, BF16), (20, 1, 128, 16, F16)])
def test_attention(ops, ragged, q_heads, kv_heads, dim, page, dtype):
    new, ctx = RAGGED[ragged]
    compare(ops, Batch(new, ctx, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page,
                       dtype=dtype, seed=1))


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype", [
    (4, 2, 80, 16, BF16), (2, 2, 256, 32, F16), (4, 2, 128, 48, BF16), (2, 1, 64, 1, F16),
    (4, 2, 128, 16, F32), (3, 3, 33, 5, F32), (2, 2, 1, 7, F32)])
@pytest.mark.parametrize("ragged", ["decode", "mixed", "empty_rows"])
def test_attention_other_shapes(ops, ragged, q_heads, kv_heads, dim, page, dtype):
    new, ctx = RAGGED[ragged]
    compare(ops, Batch(new, ctx, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page,
                       dtype=dtype, seed=2))


@pytest.mark.parametrize("ragged", ["decode", "drafts", "prompt", "mixed", "empty_rows"])
@pytest.mark.parametrize("kw", [
    dict(softcap=5.0), dict(window=1), dict(window=40), dict(window=10**6),
    dict(slopes=True), dict(prefix=[20, 1000, 0, 130, 7, 300]),
    dict(softcap=2.0, window=33, slopes=True, prefix=[3, 0, 400, 50, 0, 129]), dict(scale=0.5)],
    ids=lambda kw: "-".join(kw))
@pytest.mark.parametrize("heads,dim,dtype", [((8, 2), 128, BF16), ((3, 3), 64, F16),
                                             ((2, 1), 48, F32)])
def test_modified_scores(ops, ragged, kw, heads, dim, dtype):
    new, ctx = RAGGED[ragged]
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = 2.0 ** -torch.arange(1, heads[0] + 1).float()
    if "prefix" in kw:
        kw["prefix"] = kw["prefix"][:len(new)]
    compare(ops, Batch(new, ctx, q_heads=heads[0], kv_heads=heads[1], dim=dim, page=32,
                       dtype=dtype, seed=3), **kw)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,ctx", [([1, 1], [9000, 4100]), ([40], [7000]), ([600], [2500])])
def test_attention_split_over_a_long_context(ops, dim, new, ctx):
    compare(ops, Batch(new, ctx, q_heads=4, kv_heads=1, dim=dim, page=64, dtype=BF16, seed=4))


@pytest.mark.parametrize("dim,dtype,kw", [(128, BF16, {}), (64, F16, {}),
                                          (128, F16, dict(softcap=9.0, window=50))])
@pytest.mark.parametrize("hint", [1, 200])
def test_many_tiles_for_every_sm(ops, hint, dim, dtype, kw):
    """Short and long tiles, full and half ones, one after another."""
    new = [(7 * i * i) % 140 + 1 for i in range(40)]
    ctx = [(11 * i) % 90 if i % 3 else 0 for i in range(40)]
    compare(ops, Batch(new, ctx, q_heads=24, kv_heads=12, dim=dim, page=16, dtype=dtype, seed=10),
            hint=hint, **kw)


@pytest.mark.parametrize("kw", [{}, dict(softcap=10.0, window=100, prefix=[30, 0, 500, 64, 3, 9])])
@pytest.mark.parametrize("hint", [0, 1, 16, 100, 5000])
def test_the_hint_does_not_change_the_result(ops, hint, kw):
    new, ctx = RAGGED["mixed"]
    compare(ops, Batch(new, ctx, q_heads=8, kv_heads=2, dim=128, page=16, dtype=BF16, seed=5),
            hint=hint, **kw)


def test_large_scores_and_uniform_rows(ops):
    """Scores far apart (one key takes all) and all alike (every key the same)."""
    for factor in (0.0, 60.0):
        batch = Batch([1, 130, 3], [700, 250, 40], q_heads=8, kv_heads=2, dim=128, page=32,
                      dtype=F16, seed=6)
        batch.q = (batch.q * factor).to(F16)
        want, want_lse, spread = attend_oracle(batch)
        out, lse = attend(ops, batch)
        # fp32 scores of size s carry errors of about s 2^-20: the softmax moves by as much
        size = want_lse.abs().max().item()
        check_attention(out, None, want, None, spread * (1 + size * 2.0**-9), F16)
        assert (lse.double().cpu() - want_lse).abs().max().item() <= 2.0**-11 + size * 2.0**-18


def test_rising_scores_rescale(ops):
    """Every later key scores higher, so that the running maximum grows all along."""
    batch = Batch([1, 260], [1500, 300], q_heads=4, kv_heads=1, dim=128, page=32, dtype=BF16, seed=7)
    for b, length in enumerate(batch.seq):
        ramp = torch.linspace(-6, 6, length)[:, None]
        batch.k[b][:, 0] = (ramp * torch.ones(128)).to(BF16)
        for p in range(length):
            batch.k_cache[batch.table[b, p // 32], :, p % 32] = batch.k[b][p]
    batch.q = torch.full_like(batch.q, 1.0)
    compare(ops, batch)


def test_cache_layouts_and_strides(ops):
    """[page, slot, head, dim] storage, keys and values in one tensor, rows cut from wider ones."""
    batch = Batch([1, 60, 2], [200, 70, 33], q_heads=8, kv_heads=2, dim=128, page=32, dtype=BF16)
    want, want_lse, spread = attend_oracle(batch)
    kc, vc, table, starts, lens = batch.on(DEV)
    joint = torch.stack([kc.transpose(1, 2), vc.transpose(1, 2)], dim=1).contiguous()
    wide = torch.zeros(batch.rows, 12, 144, dtype=BF16, device=DEV)
    wide[:, 3:11, 8:136] = batch.q.to(DEV)
    for hint in (1, 60):
        out, lse = ops.paged_attention(wide[:, 3:11, 8:136], joint[:, 0].transpose(1, 2),
                                       joint[:, 1].transpose(1, 2), table, starts, lens,
                                       max_query_len=hint, return_lse=True)
        check_attention(out, lse, want, want_lse, spread, BF16)
        # operands off the 16-byte grid
        odd = torch.zeros(batch.num_pages * 2 * 32 * 128 + 1, dtype=BF16, device=DEV)[1:]
        odd = odd.view(batch.num_pages, 2, 32, 128).copy_(kc)
        q = torch.zeros(batch.rows * 8 * 128 + 1, dtype=BF16, device=DEV)[1:]
        q = q.view(batch.rows, 8, 128).copy_(batch.q)
        res = torch.zeros(batch.rows, 8, 131, dtype=BF16, device=DEV)[:, :, :128]
        for k, q_, o_ in ((odd, batch.q.to(DEV), None), (kc, q, None), (kc, q, res)):
            out, lse = ops.paged_attention(q_, k, vc, table, starts, lens, max_query_len=hint,
                                           return_lse=True, out=o_)
            check_attention(out, lse, want, want_lse, spread, BF16)
            assert o_ is None or out is o_


def test_rows_outside_every_sequence_are_zero(ops):
    for dtype, hint in ((BF16, 1), (BF16, 90), (F32, 1)):
        batch = Batch([1, 5, 1], [40, 20, 3], q_heads=4, kv_heads=2, dim=64, page=16, dtype=dtype,
                      pad_rows=130, lead_rows=2)
        out = compare(ops, batch, hint=hint)
        assert (out[:2] == 0).all() and (out[batch.starts[-1]:] == 0).all()


def test_lengths_and_tables_are_followed_no_further_than_they_reach(ops):
    """A length beyond the table's pages, page numbers out of range, starts out of order."""
    for hint in (1, 64):
        batch = Batch([1, 40], [100, 24], q_heads=4, kv_heads=2, dim=128, page=16, dtype=BF16,
                      fill=0.0)
        kc, vc, table, starts, lens = batch.on(DEV)
        q = batch.q.to(DEV)
        # sequence 0 claims more keys than the table's pages hold: the rest is not there
        far = lens.clone()
        far[0] += 10**6
        out = ops.paged_attention(q, kc, vc, table, starts, far, max_query_len=hint)
        base = ops.paged_attention(q, kc, vc, table, starts, lens, max_query_len=hint)
        assert torch.isfinite(out).all() and torch.equal(out[1:], base[1:])
        # a page number out of range reads as zeros
        bad, blank = table.clone(), kc.clone()
        bad[1, 1] = 10**6
        blank_v = vc.clone()
        blank[table[1, 1]] = 0
        blank_v[table[1, 1]] = 0
        out = ops.paged_attention(q, kc, vc, bad, starts, lens, max_query_len=hint)
        ref = ops.paged_attention(q, blank, blank_v, table, starts, lens, max_query_len=hint)
        assert torch.equal(out, ref)
        wild = torch.tensor([-5, 30, 10**9], dtype=torch.int32, device=DEV)
        assert ops.paged_attention(q, kc, vc, table, wild, lens, max_query_len=hint).shape == q.shape
    torch.cuda.synchronize()


def test_repeats_are_identical_on_any_stream(ops):
    batch = Batch([1, 300, 2], [3000, 900, 2000], q_heads=8, kv_heads=2, dim=128, page=64,
                  dtype=BF16)
    for hint in (1, 300):
        out, lse = attend(ops, batch, hint=hint)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            out2, lse2 = attend(ops, batch, hint=hint)
        side.synchronize()
        assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_graph_replay_follows_new_lengths(ops):
    """A captured step replayed with other lengths, tables and values in the same buffers."""
    first = Batch([1, 1, 1], [10, 300, 40], q_heads=8, kv_heads=2, dim=128, page=16, dtype=BF16)
    for hint in (1, 64):
        q = first.q.to(DEV)
        kc, vc, table, starts, lens = first.on(DEV)
        out = torch.empty_like(q)
        ops.paged_attention(q, kc, vc, table, starts, lens, max_query_len=hint, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(q, kc, vc, table, starts, lens, max_query_len=hint, out=out)
        second = Batch([0, 2, 1], [300, 18, 30], q_heads=8, kv_heads=2, dim=128, page=16,
                       dtype=BF16, seed=9)
        n = second.num_pages
        assert n <= first.num_pages and second.table.shape == first.table.shape
        kc[:n], vc[:n] = second.k_cache.to(DEV), second.v_cache.to(DEV)
        for dst, src in ((q, second.q), (table, second.table), (starts, second.query_start),
                         (lens, second.seq_lens)):
            dst.copy_(src)
        graph.replay()
        want, want_lse, spread = attend_oracle(second)
        check_attention(out, None, want, want_lse, spread, BF16)


def test_graphs_captured_without_a_first_call(ops):
    """Two captures on a stream that has no workspace yet: what one of them clears must not be
    needed by the other, nor by calls beside them."""
    from m5kernels_b200.linear import _workspaces

    batch = Batch([1, 1], [9000, 40], q_heads=8, kv_heads=1, dim=128, page=16, dtype=BF16)
    want, want_lse, spread = attend_oracle(batch)
    q = batch.q.to(DEV)
    args = batch.on(DEV)
    outs, graphs = [], []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    kept = {k for k in _workspaces if k[0] == "paged"}
    if any(k[-1] == side.cuda_stream for k in kept):
        pytest.skip("the stream pool handed out a used stream")
    for _ in range(2):
        out = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.paged_attention(q, *args, max_query_len=1, out=out)
        outs.append(out)
        graphs.append(graph)
    assert {k for k in _workspaces if k[0] == "paged"} == kept
    graphs[1].replay()
    torch.cuda.synchronize()
    check_attention(outs[1], None, want, want_lse, spread, BF16)
    with torch.cuda.stream(side):
        again = ops.paged_attention(q, *args, max_query_len=1)
    side.synchronize()
    check_attention(again, None, want, want_lse, spread, BF16)
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], again)


@pytest.mark.parametrize("dtype,hint", [(BF16, 1), (BF16, 64), (torch.float32, 1)])
@pytest.mark.parametrize("lens", [[40, 9000, 200], [7, 64, 3]])
def test_a_nan_query_stays_in_its_row(ops, dtype, hint, lens):
    """Its own output and lse are NaN, every other row's are as without it."""
    batch = Batch([1, 1, 2], lens, q_heads=8, kv_heads=2, dim=64, page=16, dtype=dtype)
    out, lse = attend(ops, batch, hint=hint)
    batch.q[1, 5, 3] = math.nan
    got, got_lse = attend(ops, batch, hint=hint)
    assert got[1, 5].isnan().all() and got_lse[1, 5].isnan()
    got[1, 5], got_lse[1, 5] = out[1, 5], lse[1, 5]
    assert torch.equal(got, out) and torch.equal(got_lse, lse)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hint,cap", [(1, None), (64, None), (64, 900.0)])
@pytest.mark.parametrize("faint", [18.6, 20.7])
def test_many_faint_keys_beside_a_strong_one(ops, dtype, hint, cap, faint):
    """Probabilities of 2^-faint of the largest, normal fp16 numbers only if scaled (to 2^-21): the
    strong key's values are zero, so the output is what the faint ones add up to."""
    batch = Batch([1] * 16, [1500] * 16, q_heads=8, kv_heads=8, dim=64, page=64, dtype=dtype)
    batch.q.zero_()
    batch.q[:, :, 0] = 8.0
    batch.k_cache[~batch.k_cache.isnan()] = 0.0
    batch.v_cache.abs_().add_(0.5)
    for b in range(16):
        batch.k[b].zero_()
        batch.v[b].abs_().add_(0.5)
        first = int(batch.table[b, 0])
        batch.k[b][0, :, 0] = faint * math.log(2.0)
        batch.v[b][0] = 0.0
        batch.k_cache[first, :, 0], batch.v_cache[first, :, 0] = batch.k[b][0], batch.v[b][0]
    compare(ops, batch, hint=hint, softcap=cap)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (128, BF16), (64, torch.float32)])
@pytest.mark.parametrize("page", [8, 16, 32, 128])
@pytest.mark.parametrize("prefix", [None, [10, 0, 130]])
@pytest.mark.parametrize("new,hint", [([1, 1, 1], 1), ([3, 1, 2], 3), ([1, 70, 300], 300)])
def test_pages_before_every_window_may_hold_anything(ops, dim, dtype, page, prefix, new, hint):
    """Pages that neither a prefix nor a new row's window reaches (others may own them by now)."""
    window = 100
    batch = Batch(new, [500, 259, 331], q_heads=8, kv_heads=2, dim=dim, page=page, dtype=dtype)
    for b, n in enumerate(new):
        first = -(-prefix[b] // page) if prefix else 0
        for i in range(first, (batch.seq[b] - n - window + 1) // page):
            batch.k_cache[batch.table[b, i]] = math.nan
            batch.v_cache[batch.table[b, i]] = math.inf if i % 2 else math.nan
            if i % 3 == 0:
                batch.table[b, i] = -7
    compare(ops, batch, hint=hint, window=window, prefix=prefix)


def test_offsets_beyond_32_bits(ops):
    """Pages that start more than 2^31 elements into the cache."""
    page, dim = 256, 128
    pages = (2**31 // (page * dim)) + 40
    kc = torch.empty(pages, 1, page, dim, dtype=BF16, device=DEV)
    vc = torch.empty(pages, 1, page, dim, dtype=BF16, device=DEV)
    batch = Batch([1, 140], [900, 300], q_heads=4, kv_heads=1, dim=dim, page=page, dtype=BF16)
    far = pages - batch.num_pages
    kc[far:], vc[far:] = batch.k_cache.to(DEV), batch.v_cache.to(DEV)
    table = torch.where(batch.table >= 0, batch.table + far, batch.table).to(torch.int32).to(DEV)
    want, want_lse, spread = attend_oracle(batch)
    for hint in (1, 140):
        out, lse = ops.paged_attention(batch.q.to(DEV), kc, vc, table, batch.query_start.to(DEV),
                                       batch.seq_lens.to(DEV), max_query_len=hint, return_lse=True)
        check_attention(out, lse, want, want_lse, spread, BF16)
    new = torch.randn(141, 1, dim, device=DEV).to(BF16)
    ops.paged_append(new, new, kc, vc, table, batch.query_start.to(DEV), batch.seq_lens.to(DEV))
    assert torch.equal(kc[table[0, 3], 0, 900 % page], new[0, 0])


# ---------------------------------------------------------------- appending

def tables(rows, half, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    ang = (torch.rand(rows, half, generator=g, dtype=torch.float64) * 2 - 1) * math.pi
    return torch.cos(ang).to(dtype), torch.sin(ang).to(dtype)


def check_rounded(got, want, size, dtype):
    """One rounding to the type, and three fp32 roundings of the pair's products."""
    u = UNIT[dtype]
    off = (got.double() - want).abs() - (u * want.abs() + 2.0**-22 * size + 2.0**-25)
    assert off.max().item() <= 0


@pytest.mark.parametrize("ragged", ["one", "decode", "mixed", "empty_rows"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,rot,page,x,cache,table", [
    (8, 2, 128, 128, 16, BF16, BF16, BF16), (14, 2, 64, 48, 32, F32, F16, F32),
    (4, 4, 128, 64, 64, F16, F16, F32), (3, 1, 80, 80, 7, F32, BF16, F16),
    (2, 1, 9, 6, 5, BF16, F32, F32), (4, 2, 128, 0, 16, BF16, BF16, F32),
    (56, 8, 256, 2, 128, F32, F32, F32)])
def test_append(ops, ragged, layout, q_heads, kv_heads, dim, rot, page, x, cache, table):
    new, ctx = RAGGED[ragged]
    batch = Batch(new, ctx, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, dtype=cache,
                  pad_rows=3, fill=7.0)
    g = torch.Generator().manual_seed(5)
    rows = torch.randn(batch.rows, q_heads + 2 * kv_heads, dim, generator=g).to(x)
    q, k, v = rows.split([q_heads, kv_heads, kv_heads], dim=1)
    cos, sin = tables(max(batch.seq) + 1, max(rot // 2, 1), table)
    if rot == 0:
        cos, sin = torch.ones_like(cos), torch.zeros_like(sin)
    want_k, want_v = batch.k_cache.double(), batch.v_cache.double()
    want_q = torch.zeros(q.shape, dtype=torch.float64)
    touched = torch.zeros(batch.k_cache.shape[:3], dtype=torch.bool)
    for b, (n, length) in enumerate(zip(batch.new, batch.seq)):
        for i in range(n):
            p, t = length - n + i, batch.starts[b] + i
            if p < 0:
                continue
            c, s = cos[p:p + 1], sin[p:p + 1]
            want_q[t] = rotate_oracle(q[t:t + 1], c, s, layout)[0]
            home = int(batch.table[b, p // page]), slice(None), p % page
            want_k[home] = rotate_oracle(k[t:t + 1], c, s, layout)[0]
            want_v[home] = v[t].double()
            touched[home[0], :, home[2]] = True
    gpu = rows.to(DEV)
    gq, gk, gv = gpu.split([q_heads, kv_heads, kv_heads], dim=1)
    kc, vc, tab, starts, lens = batch.on(DEV)
    kw = {} if rot == 0 else dict(cos=cos.to(DEV), sin=sin.to(DEV))
    out = ops.paged_append(gk, gv, kc, vc, tab, starts, lens, q=gq, layout=layout, **kw)
    assert out.dtype == cache and out.shape == q.shape
    check_rounded(out.cpu(), want_q, 6.0, cache)
    assert (out.cpu()[want_q == 0] == 0).all()
    for got, want, before in ((kc.cpu(), want_k, batch.k_cache), (vc.cpu(), want_v, batch.v_cache)):
        check_rounded(got[touched], want[touched], 6.0, cache)
        assert torch.equal(got[~touched], before[~touched])
    # the values are rounded once, exactly
    assert torch.equal(vc.cpu()[touched], want_v.to(x).to(cache)[touched])
    # keys and values alone leave the same cache
    kc2, vc2 = batch.on(DEV)[:2]
    assert ops.paged_append(gk, gv, kc2, vc2, tab, starts, lens, layout=layout, **kw) is None
    assert torch.equal(kc2, kc) and torch.equal(vc2, vc)


def test_append_into_other_layouts(ops):
    """[page, slot, head, dim] storage, head-major inputs, unaligned tables and rows."""
    batch = Batch([3, 50], [20, 0], q_heads=4, kv_heads=2, dim=128, page=16, dtype=BF16, fill=0.0)
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(h, batch.rows, 128, generator=g).to(BF16).to(DEV).transpose(0, 1)
               for h in (4, 2, 2))
    cos, sin = (t.to(DEV) for t in tables(80, 64, F32))
    kc, vc, tab, starts, lens = batch.on(DEV)
    want = ops.paged_append(k, v, kc, vc, tab, starts, lens, q=q, cos=cos, sin=sin)
    kt, vt = (torch.zeros(batch.num_pages, 16, 2, 129, dtype=BF16, device=DEV)[..., 1:]
              for _ in range(2))
    off = torch.zeros(80 * 64 + 1, device=DEV)
    cos2 = off[1:].view(80, 64).copy_(cos)
    flat = torch.zeros(batch.rows, 8, 130, dtype=BF16, device=DEV)
    flat[:, :, 1:129] = torch.cat([q, k, v], 1)
    q2, k2, v2 = flat[:, :, 1:129].split([4, 2, 2], dim=1)
    kt[:], vt[:] = batch.k_cache.to(DEV).transpose(1, 2), batch.v_cache.to(DEV).transpose(1, 2)
    got = ops.paged_append(k2, v2, kt.transpose(1, 2), vt.transpose(1, 2), tab, starts, lens, q=q2,
                           cos=cos2, sin=sin)
    assert torch.equal(got, want)
    assert torch.equal(kt.transpose(1, 2), kc) and torch.equal(vt.transpose(1, 2), vc)


def test_append_skips_what_has_no_place(ops):
    """Positions without a page or a table row, page numbers out of range, rows of no sequence."""
    batch = Batch([4, 2], [0, 30], q_heads=2, kv_heads=1, dim=64, page=16, dtype=BF16, fill=0.0,
                  pad_rows=5)
    x = torch.ones(batch.rows, 1, 64, dtype=BF16, device=DEV)
    q = torch.ones(batch.rows, 2, 64, dtype=BF16, device=DEV)
    kc, vc, tab, starts, lens = batch.on(DEV)
    tab = tab[:, :1].contiguous()  # positions 16.. of sequence 1 have no page
    tab[0, 0] = batch.num_pages
    cos, sin = torch.ones(31, 8, device=DEV), torch.zeros(31, 8, device=DEV)
    before = kc.clone(), vc.clone()
    out = ops.paged_append(x, x, kc, vc, tab, starts, lens, q=q, cos=cos, sin=sin)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    # tokens at 0..3 and 30 have a table row, the one at 31 and the padding have not
    assert (out[:5] == 1).all() and (out[5:] == 0).all()


# ---------------------------------------------------------------- together

def test_generation_example():
    """The quantized layer around the two operators: chunks and single tokens, mixed, against
    whole prompts.  Codes of the output projection (1/127 of a row's peak apart) may differ by one
    where two attention kernels round differently: far below 2 % of the layer's contribution."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "m5-max-kernels_b200/examples/paged_generation.py"
    spec = importlib.util.spec_from_file_location("paged_generation", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(width=1024, q_heads=8, kv_heads=2, lengths=(150, 1, 40, 97), chunk=33) < 2e-2


def test_after_the_grouped_projection(ops):
    """The head-major Q, K, V of projection_qkv_rope go into the cache without a copy."""
    g = torch.Generator().manual_seed(12)
    n, width, heads = 70, 512, 3
    x = torch.randn(n, width, generator=g).to(BF16).to(DEV)
    w = (torch.randn(heads * 384, width, generator=g) * width**-0.5).to(BF16).to(DEV)
    aq, sa = ops.quantize(x, "int8")
    bq, sb = ops.quantize(w, "int8")
    gamma = torch.ones(128, dtype=BF16, device=DEV)
    cos, sin = ops.rope_tables(n, 64, device=DEV)
    q, k, v = ops.projection_qkv_rope(aq, bq, gamma, gamma, cos, sin, "int8", a_scales=sa,
                                      b_scales=sb)
    page = 32
    kc = torch.full((4, heads, page, 128), math.nan, dtype=BF16, device=DEV)
    vc = kc.clone()
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    assert ops.paged_append(k.transpose(0, 1), v.transpose(0, 1), kc, vc, table, starts, lens) is None
    out = ops.paged_attention(q.transpose(0, 1), kc, vc, table, starts, lens, max_query_len=n)
    scores = (q.double() @ k.double().transpose(1, 2)) * 128**-0.5
    hidden = torch.ones(n, n, device=DEV).triu(1).bool()
    p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
    want, spread = (p @ v.double()).transpose(0, 1), (p @ v.double().abs()).transpose(0, 1)
    check_attention(out, None, want.cpu(), None, spread.cpu(), BF16)
