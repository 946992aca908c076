"""The paged KV cache's 8-bit form: its container and the plain PyTorch
statement of its format (any device).

A cached row (one token, one kv head, 128 dims) is held as e4m3 numbers with
one power-of-two scale: ``row = values * 2^(exps - 127)``. The exponent is the
smallest at which the row's largest magnitude is at most 448 (never below
2^-117), the values are the nearest e4m3 numbers (ties to even). A power of two
only moves exponents, so what is stored is exact in bf16 while it is below 2^128
(a row that reaches into bf16's last eighth of a binade may round up to it, a
rotated k may lie above it: infinity in bf16 and fp32). Elements that are not
finite are stored as NaN and do not take part in the maximum. A row takes 129
bytes instead of bf16's 256.
"""
import dataclasses

import torch

PAGE, HEAD_DIM = 16, 128
MIN_EXP = -117


@dataclasses.dataclass
class Fp8Pages:
    """The keys or the values of one layer: ``values`` float8_e4m3fn [blocks,
    kv heads, 16, 128] (contiguous), ``exps`` uint8 [blocks, kv heads, 16]
    (unit stride in a page, 16-byte multiples between pages). Written rows
    have bytes from 10 on; bytes 1..254 are read, exactly from 3 to 246 (1 and 2:
    some numbers lie between bf16's smallest steps; above 246: where the number
    is below 2^128). Stands wherever ``ops`` takes a bf16 ``k_cache`` /
    ``v_cache``."""
    values: torch.Tensor
    exps: torch.Tensor

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    def dequantize(self) -> torch.Tensor:
        """bf16 [blocks, kv heads, 16, 128] (plain PyTorch), as exact as the
        rows are in bf16."""
        return dequantize_rows(self.values, self.exps).to(torch.bfloat16)


def fp8_cache(num_blocks: int, kv_heads: int, device):
    """An empty 8-bit cache of one layer: (keys, values). The exponents of a
    page's keys and values share one 32-byte sector."""
    values = torch.zeros((2, num_blocks, kv_heads, PAGE, HEAD_DIM), dtype=torch.float8_e4m3fn, device=device)
    exps = torch.full((num_blocks, kv_heads, 2, PAGE), 127, dtype=torch.uint8, device=device)
    return Fp8Pages(values[0], exps[:, :, 0]), Fp8Pages(values[1], exps[:, :, 1])


def quantize_rows(x: torch.Tensor):
    """(values float8_e4m3fn, exps uint8) of rows x [..., 128] in fp32 or
    fp64: the format's definition, rounded once from x's own precision."""
    finite = torch.isfinite(x)
    m, e = torch.frexp(torch.where(finite, x, torch.zeros((), dtype=x.dtype, device=x.device)).abs().amax(-1))
    e = torch.where(m > 0.875, e - 8, e - 9)  # 448 = 0.875 * 2^9
    e = torch.where(m == 0, torch.full_like(e, MIN_EXP), e.clamp_min(MIN_EXP))
    y = torch.ldexp(x, -e.unsqueeze(-1))
    # to e4m3's four significant bits (smallest step 2^-9) at x's precision
    # first, so that fp64 rows are not rounded twice
    step = torch.frexp(y)[1].clamp_min(-5) - 4
    y = torch.ldexp(torch.round(torch.ldexp(y, -step)), step)
    y = torch.where(finite, y, torch.full((), float("nan"), dtype=x.dtype, device=x.device))
    return y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def dequantize_rows(values: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """fp32 rows of e4m3 ``values`` [..., 128] and ``exps`` [...], exact below
    2^128."""
    return torch.ldexp(values.float(), exps.to(torch.int32).unsqueeze(-1) - 127)
