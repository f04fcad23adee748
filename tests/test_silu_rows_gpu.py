"""gpu_norm_rows, SWIGLU, over the whole range of the gate, with every type of rows in and out, against silu(x) up in 64 bits.

Tolerances. f32 rows, or to f32 rows: the exponential's power is off by 2^-22.5 and the rest of its exponent by 2^-22, 1 + e^-x and the reciprocal 2^-24 and 2^-23, the rest's and
two more products 2^-24 each; below -80 two exponentials of 2^-22 each and three products: under 2^-20 of the value either way. A value below 2^-126 on the way is off by half of
2^-149 times `up`. 16-bit rows to 16-bit rows or codes: the exponent is off by 2^-24 + 2^-26.1 of itself (its rounding, and log2 e's), that is 7.4e-8 |x| of the power; with the
above 6.5e-6 + 5e-7, under 2^-17, down to -87.3; from there on 0, where the value is under 87.5 e^-87.3 = 1.05e-36."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _want(x, up):
    x, up = x.double(), up.double()
    return x / (1 + torch.exp(-x)) * up


def _gates(dt, dev):
    ends = [80.0, 87.0, 87.3, 87.33, 87.34, 87.5, 88.0, 88.7, 88.73, 89.0, 92.0, 100.0, 103.9, 104.0, 110.0, 1000.0]
    g = torch.cat([torch.linspace(-110.0, 110.0, 60001), torch.linspace(-81.0, -79.0, 2001), torch.tensor(ends), -torch.tensor(ends), torch.logspace(-30, 1, 800), -torch.logspace(-30, 1, 800)])
    return g.to(dt).to(dev)


def _rows(v, K):
    return torch.nn.functional.pad(v, (0, -v.numel() % K)).view(-1, K)


@pytest.mark.parametrize("K", [640, 16])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gates_of_every_size(pkg, dev, dtype, out, K):
    dt, odt = DT[dtype], DT[out]
    x = _rows(_gates(dt, dev), K)
    for size in (1.0, 1e4) if dt == torch.float16 else (1.0, 1e4, 1e30):
        up = (size * (1 + torch.rand(x.shape, generator=torch.Generator().manual_seed(K)))).to(dt).to(dev)
        want = _want(x, up)
        got = pkg.linear.norm_rows(torch.cat((x, up), 1), pkg.ffi.PRO_SWIGLU, K=K, up_offset=K, out_dtype=odt)
        fits = want.abs() <= torch.finfo(odt).max
        least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[odt]
        fine = torch.float32 in (dt, odt)
        bound = (torch.finfo(odt).eps / 2 + (2.0 ** -20 if fine else 2.0 ** -17)) * want.abs() + (1 + 2.0 ** -8) * (least + 2.0 ** -150 * up.double())
        if not fine:
            bound += torch.where(x.double() < -87.3, 1.05e-36 * up.double(), 0.0)
        err = (got.double() - want).abs()
        assert bool((err <= bound)[fits].all()), ((err / bound)[fits].max().item(), x[fits][(err / bound)[fits].argmax()].item())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gates_that_are_no_numbers(pkg, dev, dtype):
    """As the formula has them: silu of +inf is +inf, of -inf and NaN no number."""
    dt = DT[dtype]
    x = torch.ones(3, 128, dtype=dt, device=dev)
    x[0, 5], x[1, 6], x[2, 7] = math.inf, -math.inf, math.nan
    for out in DT.values():
        got = pkg.linear.norm_rows(torch.cat((x, torch.ones_like(x)), 1), pkg.ffi.PRO_SWIGLU, K=128, up_offset=128, out_dtype=out)
        assert float(got[0, 5]) == math.inf and math.isnan(got[1, 6]) and math.isnan(got[2, 7])
        assert int((~got.isfinite()).sum()) == 3


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scales_of_far_gates(pkg, dev, dtype):
    """e4m3: a block's scale is as exact as its largest value, here of gates from -60 to -20 with large `up`."""
    dt, K = DT[dtype], 128
    x = torch.linspace(-60.0, -20.0, 200 * K).view(200, K).flip(0).to(dt).to(dev)
    up = torch.full_like(x, 60000.0)
    codes, s = pkg.linear.norm_rows(torch.cat((x, up), 1), pkg.ffi.PRO_SWIGLU, K=K, up_offset=K, out_dtype=torch.float8_e4m3fn)
    top = _want(x, up).abs().amax(1).clamp_min(1e-30) / 448.0
    assert bool(((s[:, 0].double() - top).abs() <= ((2.0 ** -20 if dt == torch.float32 else 2.0 ** -17) + 2.0 ** -23) * top).all())
