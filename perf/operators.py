"""The paged-cache operators as measured work: appending rotated keys and values
to a paged cache, attention of new tokens over it, and the same attention with
capped, distance-biased, windowed or prefix-masked scores.

A case names one call.  The ragged lengths of its batch follow from the case
alone (`lengths`); the values and the order of the pages follow from the seed.
Token t of sequence b (rows query_start[b] .. query_start[b + 1]) stands at
position seq_lens[b] - n_b + (t - query_start[b]); seq_lens counts the new
tokens.  Position p of sequence b lives in page page_table[b, p // page], slot
p % page, of caches laid out [pages, kv heads, page, head dim].
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

_APPEND = dict(op="append", dtype="bf16", in_dtype="bf16", table="fp32", batch=1, q_heads=32,
               kv_heads=8, head_dim=128, page=64, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=0,
               lens_seed=0, layout="half", rope_dim=128)
_ATTEND = dict(op="attend", dtype="bf16", batch=1, q_heads=32, kv_heads=8, head_dim=128, page=64,
               new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=0, lens_seed=0, softcap=0.0, window=0,
               prefix=0, slopes=False, lse=False)


def listed():
    return [
        # One decoding step of a small batch writes one token a sequence: launch latency.
        dict(_APPEND, name="append_tokens", batch=24, page=16, ctx_hi=900, table="bf16"),
        # The video-length prompt (9914 rows) of the projection benchmark enters the cache at
        # once: bandwidth.
        dict(_APPEND, name="append_prompt", new_lo=9914, new_hi=9914),
        # Ragged chunks straight from an fp32 GEMM output, 64-wide heads in odd groups, adjacent
        # channels paired and only part of the head rotated, fp16 cache.
        dict(_APPEND, name="append_chunks_partial", batch=9, dtype="fp16", in_dtype="fp32",
             q_heads=14, kv_heads=2, head_dim=64, page=16, new_hi=700, ctx_hi=2000, lens_seed=3,
             layout="interleaved", rope_dim=48),
        # One user, one token, a short context: the smallest step there is.
        dict(_ATTEND, name="decode_one", ctx_lo=517, ctx_hi=517, page=16),
        # A serving batch in its decoding steady state, contexts of all lengths.
        dict(_ATTEND, name="decode_batch", batch=64, ctx_hi=8191, lens_seed=1),
        # Few users with very long contexts, wide groups: one token's work split over the GPU.
        dict(_ATTEND, name="decode_long", batch=3, q_heads=64, dtype="fp16", page=128,
             ctx_lo=60000, ctx_hi=131071, lens_seed=2),
        # A chunk of a long prompt over what is already cached, with the row statistics that
        # joining it with another part needs.
        dict(_ATTEND, name="chunk_over_cache", new_lo=512, new_hi=512, ctx_lo=16384,
             ctx_hi=16384, lse=True),
        # Two whole prompts at once: the largest call, bound by the tensor cores.
        dict(_ATTEND, name="prompt_large", batch=2, new_lo=8192, new_hi=8192, page=128),
        # Continuous batching: decoding tokens and prompt chunks of other users in one call,
        # 64-wide heads of their own keys each.
        dict(_ATTEND, name="mixed_batch", batch=20, q_heads=8, head_dim=64, dtype="fp16", page=32,
             new_hi=600, ctx_hi=3000, lens_seed=5, lse=True),
        # Prompts of a model with capped scores and a sliding window.
        dict(_ATTEND, name="capped_window_prompt", batch=3, q_heads=16, new_lo=900, new_hi=4096,
             ctx_hi=700, lens_seed=6, softcap=50.0, window=1024),
        # Its decoding step.
        dict(_ATTEND, name="capped_window_decode", batch=16, q_heads=16, ctx_lo=1, ctx_hi=8000,
             lens_seed=7, softcap=30.0, window=4096),
        # Prompts whose first part is seen by every token (an image, a question), scores falling
        # with the distance, 56 heads as in the 7168-wide projection.
        dict(_ATTEND, name="prefix_distance_prompt", batch=2, q_heads=56, kv_heads=56,
             new_lo=600, new_hi=1777, ctx_hi=90, lens_seed=8, prefix=1000, slopes=True),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm where that range is wide."""
    if hi - lo < 10:
        return rng.randint(lo, hi)
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 2))) - 1)))


@functools.lru_cache(maxsize=1)
def _limits():
    works = [work(c) for c in listed()]
    return max(w["flops"] for w in works), max(w["bytes"] for w in works)


def draw(rng: random.Random):
    """Another case of the listed ranges, no larger than the largest of them."""
    while True:
        kv = rng.choice([1, 2, 3, 4, 8, 8, 16, 56])
        group = rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
        if kv * group > 64:
            continue
        case = dict(batch=_spread(rng, 1, 96), q_heads=kv * group, kv_heads=kv,
                    head_dim=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 128, 256]),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), lens_seed=rng.randrange(1 << 20))
        ctx_hi = _spread(rng, 0, 131071)
        case.update(ctx_hi=ctx_hi, ctx_lo=rng.choice([0, ctx_hi // 2, ctx_hi]))
        # one token each, a few drafted ones, or chunks
        new_hi = rng.choice([1, 1, _spread(rng, 1, 8), _spread(rng, 8, 9914)])
        case.update(new_hi=new_hi, new_lo=rng.choice([1, new_hi]))
        if rng.random() < 0.3:
            full = dict(_APPEND, **case)
            full.update(in_dtype=rng.choice([case["dtype"], "fp32"]),
                        table=rng.choice(["fp32", "bf16"]),
                        layout=rng.choice(["half", "interleaved"]),
                        rope_dim=rng.choice([case["head_dim"], case["head_dim"] * 3 // 4, 16]))
        else:
            full = dict(_ATTEND, **case)
            full["lse"] = rng.random() < 0.3
            if rng.random() < 0.45:
                full.update(softcap=rng.choice([0.0, 20.0, 30.0, 50.0]),
                            window=rng.choice([0, _spread(rng, 16, 8192)]),
                            prefix=rng.choice([0, _spread(rng, 1, 2000)]),
                            slopes=rng.random() < 0.4)
        new, ctx = lengths(full)
        if (sum(new) + sum(ctx)) * kv * case["head_dim"] > 8 * 128 * 400_000:
            continue  # the cache of the longest listed batch
        w = work(full)
        if w["flops"] <= _limits()[0] and w["bytes"] <= _limits()[1]:
            return full


def lengths(case):
    """New tokens and cached tokens of each sequence; the first holds both upper ends."""
    rng = random.Random(case["lens_seed"])
    new, ctx = [case["new_hi"]], [case["ctx_hi"]]
    for _ in range(case["batch"] - 1):
        new.append(_spread(rng, case["new_lo"], case["new_hi"]))
        ctx.append(rng.randint(case["ctx_lo"], case["ctx_hi"]))
    return new, ctx


def prefixes(case):
    """Prefix length of each sequence: the longest, then every other one absent."""
    return [case["prefix"] * (case["batch"] - i) // case["batch"] if i % 2 == 0 else 0
            for i in range(case["batch"])]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, d, page = DTYPES[case["dtype"]], case["head_dim"], case["page"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    new, ctx = lengths(case)
    total = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    seq = [n + c for n, c in zip(new, ctx)]
    pages = [-(-s // page) for s in seq]
    count, width = sum(pages) + 3, max(pages)
    order = list(range(count))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for p in pages:
        table.append(order[at:at + p] + [-1] * (width - p))
        at += p
    state = dict(case=case, new=new, seq=seq,
                 page_table=torch.tensor(table, dtype=torch.int32, device=dev),
                 query_start=torch.tensor(starts, dtype=torch.int32, device=dev),
                 seq_lens=torch.tensor(seq, dtype=torch.int32, device=dev))
    for name in ("k_cache", "v_cache"):
        state[name] = torch.randn((count, hkv, page, d), generator=gen, device=dev, dtype=dtype)
    if case["op"] == "append":
        # the fused projection's output: query, key and value heads side by side in a row
        rows = torch.randn((total, hq + 2 * hkv, d), generator=gen, device=dev,
                           dtype=DTYPES[case["in_dtype"]])
        state["q"], state["k"], state["v"] = rows.split([hq, hkv, hkv], dim=1)
        half = case["rope_dim"] // 2
        inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        angle = torch.arange(max(seq), dtype=torch.float64, device=dev)[:, None] * inv[None, :]
        state["cos"] = torch.cos(angle).to(DTYPES[case["table"]])
        state["sin"] = torch.sin(angle).to(DTYPES[case["table"]])
    else:
        state["q"] = (1.5 * torch.randn((total, hq, d), generator=gen, device=dev)).to(dtype)
        state["slopes"] = state["prefix_lens"] = None
        if case["slopes"]:
            head = torch.arange(1, hq + 1, dtype=torch.float32, device=dev)
            state["slopes"] = torch.exp2(-8.0 * head / hq)
        if case["prefix"]:
            state["prefix"] = [min(p, s) for p, s in zip(prefixes(case), seq)]
            state["prefix_lens"] = torch.tensor(state["prefix"], dtype=torch.int32, device=dev)
        state["max_query_len"] = max(new)
    return state


@functools.lru_cache(maxsize=1)
def _framework():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "m5-max-kernels_b200"))
    import m5kernels_b200

    return m5kernels_b200


def run(state):
    if state["case"]["op"] == "append":
        return _append_own(state) if own else _append_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


def _append_own(state):
    q = _framework().paged_append(
        state["k"], state["v"], state["k_cache"], state["v_cache"], state["page_table"],
        state["query_start"], state["seq_lens"], cos=state["cos"], sin=state["sin"],
        q=state["q"], layout=state["case"]["layout"])
    return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _attend_own(state):
    case = state["case"]
    res = _framework().paged_attention(
        state["q"], state["k_cache"], state["v_cache"], state["page_table"],
        state["query_start"], state["seq_lens"], max_query_len=state["max_query_len"],
        softcap=case["softcap"] or None, window=case["window"] or None, slopes=state["slopes"],
        prefix_lens=state["prefix_lens"], return_lse=case["lse"])
    return {"out": res[0], "lse": res[1]} if case["lse"] else {"out": res}


def _append_plain(state):
    case = state["case"]
    page, half, dtype = case["page"], case["rope_dim"] // 2, DTYPES[case["dtype"]]
    token = torch.arange(state["k"].shape[0], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(state["query_start"], token, right=True) - 1
    pos = (state["seq_lens"][b] - state["query_start"][b + 1] + token).long()
    cos = state["cos"][pos].float()[:, None, :]
    sin = state["sin"][pos].float()[:, None, :]

    def rotate(x):
        x = x.float()
        turned = x.clone()
        if case["layout"] == "half":
            lo, hi = x[..., :half], x[..., half:2 * half]
            turned[..., :half] = lo * cos - hi * sin
            turned[..., half:2 * half] = hi * cos + lo * sin
        else:
            lo, hi = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            turned[..., 0:2 * half:2] = lo * cos - hi * sin
            turned[..., 1:2 * half:2] = hi * cos + lo * sin
        return turned.to(dtype)

    where = state["page_table"][b, pos // page].long()
    state["k_cache"][where, :, pos % page] = rotate(state["k"])
    state["v_cache"][where, :, pos % page] = state["v"].to(dtype)
    return {"q": rotate(state["q"]), "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _attend_plain(state):
    case = state["case"]
    q, page, d = state["q"], case["page"], case["head_dim"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    group, scale = hq // hkv, 1.0 / math.sqrt(d)
    out = torch.empty_like(q)
    lse = torch.empty((q.shape[0], hq), dtype=torch.float32, device=q.device)
    at = 0
    for i, (n, length) in enumerate(zip(state["new"], state["seq"])):
        ids = state["page_table"][i, :-(-length // page)].long()
        key = torch.arange(length, device=q.device)
        pos = torch.arange(length - n, length, device=q.device)[:, None]
        seen = key <= pos
        if case["window"]:
            seen = seen & (pos - key < case["window"])
        if case["prefix"]:
            seen = seen | (key < state["prefix"][i])
        for h in range(hkv):
            k = state["k_cache"][ids, h].reshape(-1, d)[:length].float()
            v = state["v_cache"][ids, h].reshape(-1, d)[:length].float()
            heads = slice(h * group, (h + 1) * group)
            x = torch.matmul(q[at:at + n, heads].float().transpose(0, 1), k.t()) * scale
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            if case["slopes"]:
                x = x - state["slopes"][heads, None, None] * (pos - key).abs().float()
            x = x.masked_fill(~seen, float("-inf"))
            top = x.amax(dim=-1, keepdim=True)
            p = torch.exp(x - top)
            total = p.sum(dim=-1, keepdim=True)
            out[at:at + n, heads] = (torch.matmul(p, v) / total).transpose(0, 1).to(q.dtype)
            lse[at:at + n, heads] = (top + torch.log(total))[..., 0].t()
        at += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _visible(case):
    """Per sequence: pairs of a new token and a key it sees, and keys that any token sees."""
    res = []
    for n, c, f in zip(*lengths(case), prefixes(case) if case["prefix"] else [0] * case["batch"]):
        window, f = case["window"] or (n + c), min(f, n + c)
        pairs = 0
        for p in range(c, c + n):
            lo = max(0, p + 1 - window)  # its own keys are [lo, p]
            pairs += (p + 1 - lo) + (f if f <= lo else max(f, p + 1) - (p + 1 - lo))
        first = max(0, c + 1 - window)
        res.append((pairs, n + c if f >= first else n + c - first + f))
    return res


def work(case):
    size = 2
    d, hq, hkv = case["head_dim"], case["q_heads"], case["kv_heads"]
    new, _ = lengths(case)
    total = sum(new)
    if case["op"] == "append":
        tables = 2 * case["rope_dim"] // 2 * DTYPES[case["table"]].itemsize
        values = (hq + 2 * hkv) * d
        return {"bytes": total * (values * (DTYPES[case["in_dtype"]].itemsize + size) + tables),
                "flops": total * (hq + hkv) * case["rope_dim"] * 3}
    seen = _visible(case)
    pairs, keys = sum(s[0] for s in seen), sum(s[1] for s in seen)
    return {"bytes": 2 * total * hq * d * size + 2 * keys * hkv * d * size
            + (4 * total * hq if case["lse"] else 0),
            "flops": 4 * pairs * hq * d}


def exact(case, seed):
    state = prepare(case, seed)
    new, seq = state["new"], state["seq"]
    return (_append_exact if case["op"] == "append" else _attend_exact)(case, state, new, seq)


def _append_exact(case, state, new, seq):
    """Each token as complex numbers turned by its position's angle, stored one by one."""
    r, page, d = case["rope_dim"] // 2, case["page"], case["head_dim"]
    res = {"k_cache": state["k_cache"].double(), "v_cache": state["v_cache"].double()}
    q = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    turn = torch.complex(state["cos"].double(), state["sin"].double())
    if case["layout"] == "half":
        first, second = torch.arange(r), torch.arange(r) + r
    else:
        first, second = 2 * torch.arange(r), 2 * torch.arange(r) + 1
    at = 0
    for b, (n, length) in enumerate(zip(new, seq)):
        angle = turn[length - n:length, None, :]

        def turned(x):
            x = x[at:at + n].double()
            z = torch.complex(x[..., first], x[..., second]) * angle
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q[at:at + n] = turned(state["q"])
        k, v = turned(state["k"]), state["v"][at:at + n].double()
        p = length - n
        while p < length:  # the tokens of one page at a time
            slot, i = p % page, p - (length - n)
            m = min(page - slot, length - p)
            home = int(state["page_table"][b, p // page])
            res["k_cache"][home, :, slot:slot + m] = k[i:i + m].permute(1, 0, 2)
            res["v_cache"][home, :, slot:slot + m] = v[i:i + m].permute(1, 0, 2)
            p += m
        at += n
    return {"q": q, **res}


def _attend_exact(case, state, new, seq):
    """One query head and at most 1024 tokens at a time, from the log of the sum of exponentials."""
    q, d, group = state["q"], case["head_dim"], case["q_heads"] // case["kv_heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, length) in enumerate(zip(new, seq)):
        used = (length + case["page"] - 1) // case["page"]
        home = state["page_table"][b, :used].tolist()
        keys = state["k_cache"][home].double().permute(1, 0, 2, 3).flatten(1, 2)
        vals = state["v_cache"][home].double().permute(1, 0, 2, 3).flatten(1, 2)
        for t in range(0, n, 1024):
            m = min(1024, n - t)
            far = (torch.arange(m, device="cuda").view(m, 1) + (length - n + t)
                   - torch.arange(length, device="cuda").view(1, length)).double()
            hidden = far < 0
            if case["window"]:
                hidden |= far >= case["window"]
            if case["prefix"]:
                hidden[:, :state["prefix"][b]] = False
            rows = slice(at + t, at + t + m)
            for h in range(case["q_heads"]):
                s = q[rows, h].double() @ keys[h // group, :length].mT / math.sqrt(d)
                if case["softcap"]:
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                if case["slopes"]:
                    s -= state["slopes"][h].double() * far.abs()
                s[hidden] = -math.inf
                z = torch.logsumexp(s, dim=1)
                lse[rows, h] = z
                out[rows, h] = torch.exp(s - z[:, None]) @ vals[h // group, :length]
        at += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
