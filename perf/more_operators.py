"""Block-scaled and grouped products as measured work: quantising to E4M3 with a
scale for each block of 128 channels, the matrix product of such operands, and
matrix products grouped by expert with ragged sizes.

A case names one call.  The sizes of a case's groups follow from the case alone
(`sizes`); the values follow from the seed.  Rows group_start[e] up to
group_start[e + 1] of the activations belong to expert e, whose weights are
b[e] [N, K]; both operands are K-major.  E4M3 codes are uint8, as in the
framework's quantize and gemm; where codes are an output they are returned as
the float8 values they stand for.
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128
TOP = {"fp8": 448.0, "int8": 127.0}

_QUANTIZE = dict(op="quantize", dtype="bf16", tokens=1, k=4096, copies=0, gated=False,
                 block_rows=1)
_GEMM = dict(op="gemm", out="bf16", m=1, n=4096, k=4096)
_GROUPED = dict(op="grouped", mode="fp8", scales="block", out="bf16", experts=8, tokens=1, n=4096,
                k=4096, skew=0.4, empty=0.0, behind=0, lens_seed=0)


def listed():
    return [
        # The activations of a few decoding users: launch latency.
        dict(_QUANTIZE, name="quantize_tokens", tokens=13, k=7168),
        # The input of the benchmark's FFN-down projection: bandwidth.
        dict(_QUANTIZE, name="quantize_prompt", tokens=4096, k=16384),
        # A prompt's tokens put into the order of their experts on the way, six experts a token.
        dict(_QUANTIZE, name="quantize_to_experts", tokens=1777, copies=6),
        # Between the two products of a gated FFN: the halves of one fused up-and-gate output.
        dict(_QUANTIZE, name="quantize_gated", dtype="fp16", tokens=9914, k=5376, gated=True),
        # Weights as they are loaded, a scale for each 128 x 128 block.
        dict(_QUANTIZE, name="quantize_weights", tokens=7168, k=5376, block_rows=128),
        # A projection of three decoding users: the weights are read once.
        dict(_GEMM, name="gemm_tokens", m=3, n=7168, k=5376),
        # A chunk of a prompt through FFN-down.
        dict(_GEMM, name="gemm_chunk", m=517, k=16384, out="fp16"),
        # The video-length prompt (9914 rows) through FFN-up: the largest, tensor-bound.
        dict(_GEMM, name="gemm_prompt", m=9914, n=16384),
        # Decoding: 32 users with eight experts each, a few rows for every expert.
        dict(_GROUPED, name="grouped_decode", experts=64, tokens=256, k=2048, lens_seed=1),
        # Prefill of a model with block-scaled experts.
        dict(_GROUPED, name="grouped_prompt", experts=32, tokens=32768, lens_seed=2),
        # The same of unquantised experts, large ones, one of them without tokens.
        dict(_GROUPED, name="grouped_prompt_bf16", mode="bf16", scales="none", tokens=9914, n=5376,
             empty=0.13, lens_seed=3),
        # W8A8 experts of odd widths with uneven loads, in a padded buffer, fp32 sums wanted.
        dict(_GROUPED, name="grouped_uneven_int8", mode="int8", scales="row", out="fp32",
             experts=16, tokens=2011, n=1000, k=2064, skew=1.5, empty=0.2, behind=37, lens_seed=4),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm where that range is wide."""
    if hi - lo < 10:
        return rng.randint(lo, hi)
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


@functools.lru_cache(maxsize=1)
def _limits():
    works = [work(c) for c in listed()]
    return max(w["flops"] for w in works), max(w["bytes"] for w in works)


def draw(rng: random.Random):
    """Another case of the listed ranges, no larger than the largest of them."""
    while True:
        op = rng.choice(["quantize", "gemm", "grouped", "grouped"])
        k = 16 * _spread(rng, 8, 1024)  # rows on the 16-byte grid
        if rng.random() < 0.5:
            k = max(BLOCK, k // BLOCK * BLOCK)
        n = _spread(rng, 100, 16384)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        out = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if op == "quantize":
            case = dict(_QUANTIZE, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), k=k,
                        tokens=_spread(rng, 1, 9914))
            form = rng.choice(["plain", "copies", "gated", "weights"])
            if form == "copies":
                case["copies"] = rng.randint(1, 8)
            elif form == "gated":
                case["gated"] = True
            elif form == "weights":
                case["block_rows"] = BLOCK
        elif op == "gemm":
            case = dict(_GEMM, m=_spread(rng, 1, 9914), n=n, k=k, out=out)
        else:
            mode, scales = rng.choice([("fp8", "block"), ("fp8", "block"), ("fp8", "row"),
                                       ("int8", "row"), ("bf16", "none"), ("fp16", "none")])
            case = dict(_GROUPED, mode=mode, scales=scales, out=out, n=n, k=k,
                        experts=_spread(rng, 1, 128), tokens=_spread(rng, 1, 32768),
                        skew=rng.choice([0.0, 0.4, 1.5]), empty=rng.choice([0.0, 0.2]),
                        behind=rng.choice([0, 0, rng.randint(1, 300)]),
                        lens_seed=rng.randrange(1 << 20))
            if case["experts"] * n * k > 64 * 4096 * 4096:
                continue
        w = work(case)
        if w["flops"] <= _limits()[0] and w["bytes"] <= _limits()[1]:
            return case


def sizes(case):
    """Rows of each expert: loads of a lognormal spread `skew`, some experts without any."""
    rng = random.Random(case["lens_seed"])
    load = [math.exp(rng.gauss(0.0, 1.0) * case["skew"]) for _ in range(case["experts"])]
    for e in rng.sample(range(case["experts"]), int(case["empty"] * case["experts"])):
        load[e] = 0.0
    res = [0] * case["experts"]
    for e in rng.choices(range(case["experts"]), load, k=case["tokens"]):
        res[e] += 1
    return res


def _blocks(v, block_rows):
    """v [R, K] as [R / block_rows, block_rows, K / 128, 128], padded with zeros."""
    rows, k = v.shape
    v = F.pad(v, (0, -k % BLOCK, 0, -rows % block_rows))
    return v.view(-1, block_rows, v.shape[1] // BLOCK, BLOCK)


def _quantize_blocks(v, block_rows):
    """(codes as float8 values [R, K], scales) of fp32 values."""
    rows, k = v.shape
    x = _blocks(v, block_rows)
    scale = x.abs().amax(dim=(1, 3)) / TOP["fp8"]
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = (x / scale[:, None, :, None]).clamp(-TOP["fp8"], TOP["fp8"]).to(torch.float8_e4m3fn)
    return codes.view(x.shape[0] * block_rows, -1)[:rows, :k].contiguous(), scale


def _quantize_rows(v, mode):
    """(codes, scales [R]) of fp32 values, one scale a row."""
    scale = v.abs().amax(dim=1) / TOP[mode]
    q = v / scale[:, None]
    return (q.round().to(torch.int8) if mode == "int8"
            else q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=dev, dtype=dtype)

    state, k = dict(case=case), case["k"]
    if case["op"] == "quantize":
        dtype, tokens = DTYPES[case["dtype"]], case["tokens"]
        # channels of unlike sizes, as activations have
        channel = torch.exp(0.5 * normal(k)).to(dtype)
        if case["gated"]:
            both = normal(tokens, 2 * k, dtype=dtype)
            both[:, :k] *= channel
            state["x"], state["gate"] = both[:, :k], both[:, k:]
        else:
            state["x"] = normal(tokens, k, dtype=dtype) * channel
        if case["copies"]:
            order = torch.randperm(tokens * case["copies"], generator=gen, device=dev)
            state["rows"] = (order // case["copies"]).to(torch.int32)
        return state
    if case["op"] == "gemm":
        a, state["a_scales"] = _quantize_blocks(normal(case["m"], k), 1)
        b, state["b_scales"] = _quantize_blocks(0.02 * normal(case["n"], k), BLOCK)
        state["a"], state["b"] = a.view(torch.uint8), b.view(torch.uint8)
        return state
    mode, n, experts = case["mode"], case["n"], case["experts"]
    state["sizes"] = sizes(case)
    starts = [0]
    for s in state["sizes"]:
        starts.append(starts[-1] + s)
    state["group_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    a = normal(case["tokens"] + case["behind"], k)
    if case["scales"] == "none":
        state["a"] = a.to(DTYPES[mode])
        state["b"] = 0.02 * normal(experts, n, k, dtype=DTYPES[mode])
        state["a_scales"] = state["b_scales"] = None
        return state
    quantize = (functools.partial(_quantize_rows, mode=mode) if case["scales"] == "row" else None)
    weights, scales = [], []
    if quantize is None:
        a, state["a_scales"] = _quantize_blocks(a, 1)
        state["a"] = a.view(torch.uint8)
    else:
        state["a"], state["a_scales"] = quantize(a)
    for _ in range(experts):
        w = 0.02 * normal(n, k)
        q, s = _quantize_blocks(w, BLOCK) if quantize is None else quantize(w)
        weights.append(q.view(torch.uint8) if quantize is None else q)
        scales.append(s)
    state["b"], state["b_scales"] = torch.stack(weights), torch.stack(scales)
    return state


@functools.lru_cache(maxsize=1)
def _framework():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "m5-max-kernels_b200"))
    import m5kernels_b200

    return m5kernels_b200


def run(state):
    op = state["case"]["op"]
    if op == "quantize":
        return _quantize_own(state) if own else _quantize_plain(state)
    if op == "gemm":
        return _gemm_own(state) if own else _gemm_plain(state)
    return _grouped_own(state) if own else _grouped_plain(state)


def _quantize_own(state):
    codes, scales = _framework().block_quantize(
        state["x"], gate=state.get("gate"), rows=state.get("rows"),
        block_rows=state["case"]["block_rows"])
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales}


def _gemm_own(state):
    return {"out": _framework().block_gemm(
        state["a"], state["b"], state["a_scales"], state["b_scales"],
        output_dtype=DTYPES[state["case"]["out"]])}


def _grouped_own(state):
    case = state["case"]
    return {"out": _framework().grouped_gemm(
        state["a"], state["b"], state["group_start"], case["mode"], a_scales=state["a_scales"],
        b_scales=state["b_scales"], output_dtype=DTYPES[case["out"]])}


def _quantize_plain(state):
    x = state["x"]
    if "rows" in state:
        x = x[state["rows"].long()]
    v = x.float()
    if "gate" in state:
        g = state["gate"].float()
        v = g / (1.0 + torch.exp(-g)) * v
    codes, scales = _quantize_blocks(v, state["case"]["block_rows"])
    return {"codes": codes, "scales": scales}


def _values(codes, scales, block_rows):
    """Block-scaled E4M3 codes [R, K] as fp32."""
    x = _blocks(codes.view(torch.float8_e4m3fn).float(), block_rows) * scales[:, None, :, None]
    return x.view(x.shape[0] * block_rows, -1)[:codes.shape[0], :codes.shape[1]]


def _gemm_plain(state):
    a = _values(state["a"], state["a_scales"], 1)
    b = _values(state["b"], state["b_scales"], BLOCK)
    return {"out": torch.matmul(a, b.t()).to(DTYPES[state["case"]["out"]])}


def _grouped_plain(state):
    case, a, b = state["case"], state["a"], state["b"]
    sa, sb = state["a_scales"], state["b_scales"]
    out = torch.zeros((a.shape[0], case["n"]), dtype=DTYPES[case["out"]], device=a.device)
    at = 0
    for e, rows in enumerate(state["sizes"]):
        if rows == 0:
            continue
        mine = slice(at, at + rows)
        if case["scales"] == "block":
            y = torch.matmul(_values(a[mine], sa[mine], 1), _values(b[e], sb[e], BLOCK).t())
        elif case["scales"] == "none":
            y = torch.matmul(a[mine].float(), b[e].float().t())
        elif case["mode"] == "fp8":
            y = torch.matmul(a[mine].view(torch.float8_e4m3fn).float(),
                             b[e].view(torch.float8_e4m3fn).float().t())
            y = y * sa[mine, None] * sb[e]
        else:  # sums of whole numbers that fp32 does not hold
            y = torch.matmul(a[mine].double(), b[e].double().t()).float()
            y = y * sa[mine, None] * sb[e]
        out[mine] = y.to(out.dtype)
        at += rows
    return {"out": out}


def work(case):
    k = case["k"]
    groups = -(-k // BLOCK)
    if case["op"] == "quantize":
        rows = case["tokens"] * max(1, case["copies"])
        read = case["tokens"] * k * DTYPES[case["dtype"]].itemsize * (2 if case["gated"] else 1)
        scales = -(-rows // case["block_rows"]) * groups
        return {"bytes": read + rows * k + 4 * scales + (4 * rows if case["copies"] else 0),
                "flops": rows * k * (8 if case["gated"] else 3)}
    out = DTYPES[case["out"]].itemsize
    if case["op"] == "gemm":
        m, n = case["m"], case["n"]
        return {"bytes": m * k + n * k + out * m * n + 4 * groups * (m + -(-n // BLOCK)),
                "flops": 2 * m * n * k}
    size = 2 if case["scales"] == "none" else 1
    rows, n = case["tokens"], case["n"]
    busy = sum(1 for s in sizes(case) if s)
    scales = {"none": 0, "row": 4 * (rows + busy * n),
              "block": 4 * groups * (rows + busy * -(-n // BLOCK))}[case["scales"]]
    return {"bytes": (rows + busy * n) * k * size + out * (rows + case["behind"]) * n + scales
            + 4 * (case["experts"] + 1),
            "flops": 2 * rows * n * k}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _quantize_exact(case, state)
    if case["op"] == "gemm":
        return {"out": _product_exact(state["a"], state["b"], state["a_scales"],
                                      state["b_scales"])}
    out = torch.zeros((state["a"].shape[0], case["n"]), dtype=torch.float64, device="cuda")
    bounds = state["group_start"].tolist()
    for e in range(case["experts"]):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        a, b = state["a"][lo:hi], state["b"][e]
        if case["scales"] == "block":
            out[lo:hi] = _product_exact(a, b, state["a_scales"][lo:hi], state["b_scales"][e])
            continue
        if case["mode"] == "fp8":
            a, b = a.view(torch.float8_e4m3fn), b.view(torch.float8_e4m3fn)
        out[lo:hi] = a.double() @ b.double().mT
        if case["scales"] == "row":
            out[lo:hi] *= torch.outer(state["a_scales"][lo:hi].double(),
                                      state["b_scales"][e].double())
    return {"out": out}


def _product_exact(a, b, a_scales, b_scales):
    """The sum over the blocks of 128 channels of their products times their scales."""
    k = a.shape[1]
    out = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.float64, device="cuda")
    for g in range(a_scales.shape[1]):
        at = slice(g * BLOCK, min(k, (g + 1) * BLOCK))
        x = a[:, at].view(torch.float8_e4m3fn).double()
        w = b[:, at].view(torch.float8_e4m3fn).double()
        scale = b_scales[:, g].double().repeat_interleave(BLOCK)[:b.shape[0]]
        out += (x @ w.mT) * a_scales[:, g, None].double() * scale
    return out


def _quantize_exact(case, state):
    """Codes as the multiples of 2^(exponent - 3) next to the quotient, ties to even.  Scales are
    fp32 numbers and so, by the definition that quantize has too, is the quotient."""
    v = state["x"].double()
    if case["gated"]:
        v = v * state["gate"].double() * torch.sigmoid(state["gate"].double())
    rows, k = v.shape
    step = case["block_rows"]
    codes = torch.empty((rows, k), dtype=torch.float64, device="cuda")
    scales = torch.empty((-(-rows // step), -(-k // BLOCK)), dtype=torch.float64, device="cuda")
    for g in range(scales.shape[1]):
        at = slice(g * BLOCK, min(k, (g + 1) * BLOCK))
        peak = v[:, at].abs().max(dim=1).values
        if step > 1:
            peak = torch.stack([p.max() for p in peak.split(step)])
        scales[:, g] = torch.where(peak > 0, peak / 448.0, 1.0)
        held = scales[:, g].float().double().repeat_interleave(step)[:rows, None]
        q = (v[:, at] / held).float().double()
        unit = torch.exp2(torch.frexp(q)[1].double().sub(1.0).clamp(min=-6.0) - 3.0)
        codes[:, at] = (torch.round(q / unit) * unit).clamp(-448.0, 448.0)
    if case["copies"]:
        rows = state["rows"].long()
        codes, scales = codes[rows], scales[rows]
    return {"codes": codes, "scales": scales}
