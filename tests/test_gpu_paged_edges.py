"""The paged cache where it went wrong once: workspaces of graphs, extreme scores and positions."""

import pytest
import torch

from paged_cases import Batch, attend_oracle, check_attention

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m
    from m5kernels_b200 import _lib

    yield m
    assert _lib.device_status() == 0  # no bounded wait gave up


# ---------------------------------------------------------------- workspaces

@pytest.mark.parametrize("hint", [1, 64])
def test_a_graph_keeps_its_workspace(ops, hint):
    """A stream's workspace is replaced by a larger one after a graph was captured there."""
    batch = Batch([1, 1], [9000, 40], q_heads=8, kv_heads=1, dim=64, page=16, dtype=BF16)
    wide = Batch([1, 1], [9000, 40], q_heads=8, kv_heads=1, dim=128, page=16, dtype=BF16)
    want, want_lse, spread = attend_oracle(batch)
    q, args = batch.q.to(DEV), batch.on(DEV)
    wide_q, wide_args = wide.q.to(DEV), wide.on(DEV)
    out, graph, side = torch.empty_like(q), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        first = ops.paged_attention(q, *args, max_query_len=hint)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        ops.paged_attention(q, *args, max_query_len=hint, out=out)
    with torch.cuda.stream(side):
        ops.paged_attention(wide_q, *wide_args, max_query_len=hint)
        taken = [torch.full((1 << 20,), i, dtype=torch.int32, device=DEV) for i in range(32)]
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    check_attention(out, None, want, want_lse, spread, BF16)
    assert torch.equal(out, first)
    assert all((t == i).all() for i, t in enumerate(taken))


def test_graphs_replayed_beside_each_other(ops):
    """Two graphs captured on one stream, and that stream's own calls, on three streams at once."""
    batch = Batch([1, 1], [9000, 40], q_heads=8, kv_heads=1, dim=128, page=16, dtype=BF16)
    q, args = batch.q.to(DEV), batch.on(DEV)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        want = ops.paged_attention(q, *args, max_query_len=1)
    torch.cuda.synchronize()
    outs, graphs = [], []
    for _ in range(2):
        out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            for _ in range(3):
                ops.paged_attention(q, *args, max_query_len=1, out=out)
        outs.append(out)
        graphs.append(graph)
    for _ in range(20):
        for graph, stream in zip(graphs, streams[1:]):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[0]):
            got = ops.paged_attention(q, *args, max_query_len=1)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(out, want) for out in outs)


# ---------------------------------------------------------------- NaN and infinities

KINDS = [(64, BF16, 64), (128, F16, 64), (128, BF16, 1), (64, F32, 1)]  # prompt, decode, row kernel


def attend(ops, batch, hint, **kw):
    return ops.paged_attention(batch.q.to(DEV), *batch.on(DEV), max_query_len=hint, return_lse=True,
                               **kw)


def check_nan_rows(got, clean, rows, heads):
    """The named rows and heads are NaN, all others as they were."""
    for x, y in zip(got, clean):
        assert x[rows][:, heads].isnan().all()
        x[rows, heads] = y[rows, heads]
        assert torch.equal(x, y)


@pytest.mark.parametrize("dim,dtype,hint", KINDS)
@pytest.mark.parametrize("window", [None, 3])
def test_a_nan_query_at_any_position(ops, dim, dtype, hint, window):
    """Whichever keys the row sees, however few: its out and lse are NaN, no other's."""
    batch = Batch([21, 2], [0, 40], q_heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    clean = attend(ops, batch, hint, window=window)
    for at in range(21):
        batch.q[at, 1, 5], kept = float("nan"), batch.q[at, 1, 5].clone()
        check_nan_rows(attend(ops, batch, hint, window=window), clean, slice(at, at + 1), slice(1, 2))
        batch.q[at, 1, 5] = kept


@pytest.mark.parametrize("dim,dtype,hint", KINDS)
@pytest.mark.parametrize("value", ["nan", "overflow"])
def test_a_nan_or_infinite_score_reaches_its_rows(ops, dim, dtype, hint, value):
    """A key at each slot of a block, NaN or so large that the score overflows to +inf: the rows
    that see it are NaN, as the softmax of such scores is."""
    if value == "overflow" and dtype is F16:
        pytest.skip("fp16 products do not overflow fp32")
    batch = Batch([70, 2], [0, 40], q_heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    batch.q[:, :, 0] = 1.0 if value == "nan" else 1e30
    batch.k_cache[..., 0] = 0.0
    clean = attend(ops, batch, hint)
    for slot in range(64):
        home = int(batch.table[0, slot // 16]), 1, slot % 16, 0
        batch.k_cache[home] = float("nan") if value == "nan" else 1e30
        check_nan_rows(attend(ops, batch, hint), clean, slice(slot, 70), slice(2, 4))
        batch.k_cache[home] = 0.0


# ---------------------------------------------------------------- precision

@pytest.mark.parametrize("dim,dtype,hint", [(64, BF16, 300), (128, BF16, 300), (128, F16, 300),
                                            (64, BF16, 1), (128, F16, 1), (128, F32, 300)])
@pytest.mark.parametrize("kw", [{}, dict(window=1), dict(window=5), dict(scale=0.01)],
                         ids=lambda kw: "-".join(f"{k}{v}" for k, v in kw.items()) or "plain")
def test_lse_has_the_precision_of_its_type(ops, dim, dtype, hint, kw):
    """The products of 16-bit inputs are exact in fp32, in which scores, exponentials and sums are
    held whatever the cache's type: 2^-16 for those and 2^-20 of the logarithm itself, as for an
    fp32 cache."""
    batch = Batch([300, 3], [0, 200], q_heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    want = attend_oracle(batch, **kw)[1]
    lse = attend(ops, batch, hint, **kw)[1].double().cpu()
    assert ((lse - want).abs() - (2.0**-16 + 2.0**-20 * want.abs())).max().item() <= 0


@pytest.mark.parametrize("dim,dtype,hint", KINDS)
@pytest.mark.parametrize("kw", [{}, dict(window=40), dict(softcap=30.0)],
                         ids=lambda kw: "-".join(kw) or "plain")
def test_hidden_keys_weigh_nothing(ops, dim, dtype, hint, kw):
    """Values of hidden keys as large as the type holds do not move a row by a bit."""
    large = 60000.0 if dtype is F16 else 3e38
    batch = Batch([150, 1], [30, 40], q_heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    clean = attend(ops, batch, hint, **kw)
    for key in (33, 90, 134, 179):  # positions 30 .. 179 are new rows
        home = int(batch.table[0, key // 16]), slice(None), key % 16
        kept = batch.v_cache[home].clone()
        batch.v_cache[home] = large
        got = attend(ops, batch, hint, **kw)
        seen = torch.zeros(151, dtype=torch.bool)
        seen[key - 30:min(150, key - 30 + kw.get("window", 1000))] = True
        assert torch.equal(got[0].cpu()[~seen], clean[0].cpu()[~seen])
        assert torch.equal(got[1], clean[1])
        batch.v_cache[home] = kept


@pytest.mark.parametrize("dim,dtype,hint", [(64, BF16, 64), (128, F16, 64), (128, BF16, 1),
                                            (64, F16, 1), (64, F32, 1)])
@pytest.mark.parametrize("cap", [3.0, 900.0, 1e3, 1e4, 1e5, 1e6, 1e8, 1e30])
def test_large_caps(ops, dim, dtype, hint, cap):
    """A cap far above the scores changes next to nothing, in every kernel: scores are off by
    2^-16 at most (check_attention's e for fp32), not by a share of the cap."""
    batch = Batch([1, 70, 2], [200, 30, 500], q_heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype)
    want, want_lse, spread = attend_oracle(batch, softcap=cap)
    out, lse = attend(ops, batch, hint, softcap=cap)
    check_attention(out, lse, want, want_lse, spread, dtype)
    off = (lse.double().cpu() - want_lse).abs()
    assert (off - (2.0**-16 + 2.0**-20 * want_lse.abs())).max().item() <= 0


@pytest.mark.parametrize("dim,dtype,hint", [(64, BF16, 64), (128, F16, 64), (128, BF16, 1)])
@pytest.mark.parametrize("cap", [1e3, 1e5])
def test_scores_on_both_sides_of_a_large_cap(ops, dim, dtype, hint, cap):
    """Ordinary rows beside ones whose scores exceed the cap: 2^-16 for the scores of the former
    as without those; the others' scores are of the cap's size and off by the 2^-20 of it that tanh
    has and a few fp32 roundings, 2^-19 together."""
    batch = Batch([70, 2], [60, 500], q_heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype)
    batch.q[::3] *= 60000.0 / batch.q.abs().max()  # (within fp16)
    scale = 2 * cap / 60000.0 if cap > 1e4 else dim ** -0.5
    batch.q[1::3] *= dim ** -0.5 / scale if cap > 1e4 else 1.0
    batch.q[2::3] *= dim ** -0.5 / scale if cap > 1e4 else 1.0
    want, want_lse, _ = attend_oracle(batch, softcap=cap, scale=scale)
    lse = attend(ops, batch, hint, softcap=cap, scale=scale)[1].double().cpu()
    large = torch.zeros(72, dtype=torch.bool)
    large[::3] = True
    assert want_lse[large].max().item() > 0.7 * cap
    off = (lse - want_lse).abs() - (2.0**-16 + 2.0**-20 * want_lse.abs())
    assert off[~large].max().item() <= 0 and want_lse[~large].abs().max().item() < 100
    assert (lse - want_lse)[large].abs().max().item() <= 2.0**-19 * cap


@pytest.mark.parametrize("dim,hint", [(64, 64), (128, 64), (128, 1)])
@pytest.mark.parametrize("cap,scale,size", [(1e30, 1.0, 1e12), (1e37, 0.125, 1e12),
                                            (1.5e-38, 8.0, 1.0), (1e-30, 1e20, 1e-3)])
def test_caps_and_scores_at_the_ends_of_the_range(ops, dim, hint, cap, scale, size):
    """Squares and ratios of them that fp32 does not hold: no NaN, and the softmax is right."""
    batch = Batch([70, 2], [60, 300], q_heads=4, kv_heads=2, dim=dim, page=16, dtype=BF16)
    batch.q *= size
    batch.q[3] = 0.0  # scores of zero
    for b in range(2):
        batch.k[b] *= size if size > 1.0 else 1.0
    batch.k_cache *= size if size > 1.0 else 1.0
    want, want_lse, spread = attend_oracle(batch, softcap=cap, scale=scale)
    out, lse = attend(ops, batch, hint, softcap=cap, scale=scale)
    if cap < 1.0:  # scores next to zero: every key weighs the same
        check_attention(out, lse, want, want_lse, spread, BF16)
    else:  # one key takes all, unless two are within fp32's rounding of one another
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        assert ((lse.double().cpu() - want_lse).abs() <= 2.0**-18 * want_lse.abs() + 2.0**-16).all()


# ---------------------------------------------------------------- positions

@pytest.mark.parametrize("dim,dtype,hint", KINDS)
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("page", [16, 256])
def test_the_last_positions_of_32_bits(ops, dim, dtype, hint, new, page):
    """A sequence of 2^31 - 1 tokens, of which a window sees the last ones."""
    length = 2 * page - 1 + (512 if page == 16 else 0)
    batch = Batch([new], [length - new], q_heads=4, kv_heads=2, dim=dim, page=page, dtype=dtype)
    want, want_lse, spread = attend_oracle(batch, window=100)
    kc, vc, table, starts, lens = batch.on(DEV)
    far = torch.full((1, 2**31 // page), -1, dtype=torch.int32, device=DEV)
    far[:, -table.shape[1]:] = table
    lens.fill_(2**31 - 1)
    out, lse = ops.paged_attention(batch.q.to(DEV), kc, vc, far, starts, lens, max_query_len=hint,
                                   window=100, return_lse=True)
    check_attention(out, lse, want, want_lse, spread, dtype)
    rows = torch.randn(new, 2, dim, device=DEV).to(dtype)
    ops.paged_append(rows, rows, kc, vc, far, starts, lens)
    at = torch.arange(length - new, length, device=DEV)
    where = table[0, at // page].long()
    assert torch.equal(kc[where, :, at % page], rows) and torch.equal(vc[where, :, at % page], rows)


@pytest.mark.parametrize("far", [2**31, 10**30])
def test_windows_and_hints_of_any_size(ops, far):
    batch = Batch([1, 70], [200, 30], q_heads=4, kv_heads=2, dim=64, page=16, dtype=BF16)
    want, want_lse, spread = attend_oracle(batch)
    out, lse = attend(ops, batch, far, window=far)
    check_attention(out, lse, want, want_lse, spread, BF16)


@pytest.mark.parametrize("dim,dtype,hint", KINDS)
@pytest.mark.parametrize("cap", [None, 5.0, 50.0, 500.0])
def test_other_sequences_do_not_move_a_bit(ops, dim, dtype, hint, cap):
    """Whatever their queries and keys are, on both sides of the cap."""
    batch = Batch([70, 30], [60, 75], q_heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype)
    clean = attend(ops, batch, hint, softcap=cap)
    batch.q[70:] *= 100.0
    batch.k_cache[batch.table[1, :4].long()] *= 100.0
    got = attend(ops, batch, hint, softcap=cap)
    for x, y in zip(got, clean):
        assert torch.equal(x[:70], y[:70]) and not torch.equal(x[70:], y[70:])


@pytest.mark.parametrize("dim,dtype,hint", KINDS)
@pytest.mark.parametrize("cap", [None, 5.0, 50.0, 500.0])
@pytest.mark.parametrize("new,ctx", [([70, 30], [60, 75]), ([1, 64, 65, 200], [3, 0, 0, 7])])
def test_unused_slots_do_not_move_a_bit(ops, dim, dtype, hint, cap, new, ctx):
    """Whatever the slots behind the sequences' ends hold."""
    batch = Batch(new, ctx, q_heads=4, kv_heads=2, dim=dim, page=16, dtype=dtype, fill=0.0)
    clean = attend(ops, batch, hint, softcap=cap)
    for held in (1000.0, float("inf"), float("nan")):
        for b, end in enumerate(batch.seq):
            if end % 16:
                batch.k_cache[batch.table[b, end // 16], :, end % 16:] = held
                batch.v_cache[batch.table[b, end // 16], :, end % 16:] = held
        assert all(torch.equal(x, y) for x, y in zip(attend(ops, batch, hint, softcap=cap), clean))


# ---------------------------------------------------------------- the ring

@pytest.mark.parametrize("dim,dtype,page,window", [(128, F16, 64, None), (128, BF16, 64, 500),
                                                   (128, BF16, 16, None), (64, F16, 64, None)])
def test_copies_out_of_l2_wait_for_the_last_reads(ops, dim, dtype, page, window):
    """Many row tiles over the same keys in the decode kernel, whose copies then come out of L2 and
    follow a stage's release at once: each of 20 calls gives the same, and the right, result."""
    kv, group = 4, 4
    g = torch.Generator().manual_seed(11)
    new = [1 + int(n) for n in torch.randint(0, 300, (30,), generator=g)]
    new[::2] = [1] * 15
    seq = [n + int(c) for n, c in zip(new, torch.randint(0, 4000, (30,), generator=g))]
    pages = [-(-s // page) for s in seq]
    order = torch.randperm(sum(pages), generator=g).split(pages)
    table = torch.nn.utils.rnn.pad_sequence([o.to(torch.int32) for o in order], True, -1).to(DEV)
    make = lambda *shape: torch.randn(*shape, generator=g).to(dtype).to(DEV)
    kc, vc = (make(sum(pages), kv, page, dim) for _ in range(2))
    q = make(sum(new), kv * group, dim)
    starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
    lens = torch.tensor(seq, dtype=torch.int32, device=DEV)
    runs = [ops.paged_attention(q, kc, vc, table, starts, lens, max_query_len=1, window=window,
                                return_lse=True) for _ in range(20)]
    for out, lse in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(lse, runs[0][1])
    want, spread = (torch.empty(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    want_lse = torch.empty(q.shape[:2], dtype=torch.float64, device=DEV)
    for b, (n, length) in enumerate(zip(new, seq)):
        k, v = (c[order[b].to(DEV)].transpose(0, 1).flatten(1, 2)[:, :length].double()
                .repeat_interleave(group, 0) for c in (kc, vc))
        rows = slice(int(starts[b]), int(starts[b]) + n)
        x = q[rows].double().transpose(0, 1) @ k.transpose(1, 2) * dim ** -0.5
        far = (torch.arange(length - n, length, device=DEV)[:, None]
               - torch.arange(length, device=DEV)[None, :])
        x = x.masked_fill((far < 0) | (far >= (window or length)), float("-inf"))
        p = torch.softmax(x, -1)
        want[rows], spread[rows] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
        want_lse[rows] = torch.logsumexp(x, -1).t()
    check_attention(runs[0][0], runs[0][1], want.cpu(), want_lse.cpu(), spread.cpu(), dtype)
