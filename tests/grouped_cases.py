"""Operands of the block-scaled and grouped products for the tests, and their 64-bit oracles."""

import torch

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128


def blocks(v, block_rows):
    """v [R, K] as [R / block_rows, block_rows, K / 128, 128], padded with zeros."""
    rows, k = v.shape
    v = torch.nn.functional.pad(v, (0, -k % BLOCK, 0, -rows % block_rows))
    return v.view(-1, block_rows, v.shape[1] // BLOCK, BLOCK)


def e4m3_round(q):
    """The E4M3 value next to each fp64 value, ties to even, saturating at 448."""
    unit = torch.exp2(torch.frexp(q)[1].double().sub(1.0).clamp(min=-6.0) - 3.0)
    return (torch.round(q / unit) * unit).clamp(-448.0, 448.0)


def quantize_oracle(v, block_rows=1):
    """(values of the codes in 64 bits, fp32 scales) of fp32 values v [R, K].

    The scale and the quotient are fp32 operations: computed in 64 bits and
    rounded once (a quotient of fp32 numbers needs no more than 50).
    """
    rows, k = v.shape
    x = blocks(v.double(), block_rows)
    scale = (x.abs().amax(dim=(1, 3)) / 448.0).float()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = e4m3_round((x / scale.double()[:, None, :, None]).float().double())
    return q.reshape(x.shape[0] * block_rows, x.shape[2] * BLOCK)[:rows, :k], scale


def values(codes):
    """uint8 E4M3 codes as fp64 values."""
    return codes.view(torch.float8_e4m3fn).float().double()


def dequantized(codes, scales, block_rows):
    x = blocks(values(codes), block_rows) * scales.double()[:, None, :, None]
    return x.reshape(x.shape[0] * block_rows, x.shape[2] * BLOCK)[:codes.shape[0], :codes.shape[1]]


class Experts:
    """Grouped operands on the CPU: sizes of the groups, `lead` rows before the first and
    `behind` after the last, which hold NaN where the type has it."""

    def __init__(self, sizes, *, n, k, mode, scales="none", lead=0, behind=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.sizes, self.n, self.k, self.mode, self.scales = list(sizes), n, k, mode, scales
        starts = [lead]
        for s in sizes:
            starts.append(starts[-1] + s)
        self.starts, self.rows = starts, starts[-1] + behind
        self.group_start = torch.tensor(starts, dtype=torch.int32)
        experts, kb = len(sizes), -(-k // BLOCK)
        if mode == "int8":
            self.a = torch.randint(-127, 128, (self.rows, k), generator=g).to(torch.int8)
            self.b = torch.randint(-127, 128, (experts, n, k), generator=g).to(torch.int8)
        elif mode == "fp8":
            def codes(*shape):
                v = (3.0 * torch.randn(shape, generator=g)).to(torch.float8_e4m3fn)
                return v.view(torch.uint8)

            self.a, self.b = codes(self.rows, k), codes(experts, n, k)
        else:
            self.a = torch.randn(self.rows, k, generator=g).to(DTYPE[mode])
            self.b = torch.randn(experts, n, k, generator=g).to(DTYPE[mode])
        outside = torch.ones(self.rows, dtype=torch.bool)
        outside[starts[0]:starts[-1]] = False
        if mode == "fp8":
            self.a[outside] = 0x7F
        elif mode != "int8":
            self.a[outside] = float("nan")
        self.outside = outside
        self.a_scales = self.b_scales = None

        def positive(*shape):  # (over a few powers of two)
            return torch.exp2(4.0 * torch.rand(shape, generator=g) - 8.0)

        if scales == "row":
            self.a_scales, self.b_scales = positive(self.rows), positive(experts, n)
        elif scales == "block":
            self.a_scales = positive(self.rows, kb)
            self.b_scales = positive(experts, -(-n // BLOCK), kb)

    def on(self, dev):
        """The arguments of grouped_gemm."""
        move = lambda t: None if t is None else t.to(dev)  # noqa: E731
        return dict(a=move(self.a), b=move(self.b), group_start=move(self.group_start),
                    mode=self.mode, a_scales=move(self.a_scales), b_scales=move(self.b_scales))

    def oracle(self):
        """(out, spread) in 64 bits: spread = the sum of the terms' magnitudes."""
        out = torch.zeros(self.rows, self.n, dtype=torch.float64)
        spread = torch.zeros_like(out)
        for e in range(len(self.sizes)):
            mine = slice(self.starts[e], self.starts[e + 1])
            a, b = self.a[mine], self.b[e]
            if self.scales == "block":
                a = dequantized(a, self.a_scales[mine], 1)
                b = dequantized(b, self.b_scales[e], BLOCK)
            else:
                a = values(a) if self.mode == "fp8" else a.double()
                b = values(b) if self.mode == "fp8" else b.double()
                if self.scales == "row":
                    a = a * self.a_scales[mine, None].double()
                    b = b * self.b_scales[e][:, None].double()
            out[mine], spread[mine] = a @ b.T, a.abs() @ b.abs().T
        return out, spread


def check_product(got, out, spread, k):
    """|error| <= u |out| + e sum |terms|.

    u rounds the output.  Each of the at most ceil(K / 16) matrix instructions
    of a sum, and each of its ceil(K / 128) scaled additions, is off by at most
    2^-22 of the sum of magnitudes (an fp32 accumulator that may truncate), and
    three fp32 products by scales by 2^-24 each: e = (K / 16 + K / 128 + 3) 2^-22.
    """
    u = UNIT[got.dtype]
    e = (-(-k // 16) + -(-k // 128) + 3) * 2.0**-22
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    excess = (got - out).abs() - (u * out.abs() + (1 + u) * e * spread + 2.0**-133)
    assert excess.max().item() <= 0, excess.max().item()
