"""gpu_packed_attention where a CTA goes through more items than there are places for its notes of numbers that are none (eight, csrc/attention_tc.cu): what a row does not see does
not reach it, in whichever of the CTA's items it comes."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


# Items of a CTA: rows / tokens of an item, times groups of heads, over 148 SMs. At most 32 sequences come by length, more of them in their own order with tiles that nobody needs
# in between; items of one key tile and of many, with a second tile and without
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D,lens", [(64, 64, 64, [1, 300, 40, 700, 256, 257, 0, 5, 129, 1000] * 3), (64, 64, 64, [130, 2, 0, 400, 77] * 16),
                                          (64, 8, 128, [2500, 33, 31, 700, 1, 64, 90] * 4), (128, 4, 128, [9, 500, 0, 130] * 12), (96, 96, 40, [90] * 40 + [600] * 8)])
def test_notes_of_many_items(pkg, dev, H, Hkv, D, lens, dtype):
    g = torch.Generator().manual_seed(H + D + len(lens))
    dt = torch.float16 if dtype == "f16" else torch.bfloat16
    o = [0]
    for n in lens:
        o.append(o[-1] + n)
    rows, ratio = o[-1], H // Hkv
    tokens = 256 // min(ratio, 16)
    items = sum(-(-n // tokens) for n in lens) * (H // min(ratio, 16))
    assert items > 16 * torch.cuda.get_device_properties(dev).multi_processor_count
    q, k, v = ((torch.randn(rows, h, D, generator=g) * s).to(dt).to(dev) for h, s in ((H, 2.0), (Hkv, 1.5), (Hkv, 1.0)))
    offsets = torch.tensor(o, dtype=torch.int32, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))          # of each row
    end = torch.tensor(o[1:])[seq]
    clean = pkg.attention.packed_attention(q, k, v, offsets)
    assert torch.equal(pkg.attention.packed_attention(q, k, v, offsets), clean)
    for many in (1, 20, 400):
        bad = v.clone()
        fine = torch.ones(rows, H, D, dtype=torch.bool, device=dev)
        for n in range(many):
            row, head, column = int(torch.randint(rows, (1,), generator=g)), int(torch.randint(Hkv, (1,), generator=g)), int(torch.randint(D, (1,), generator=g))
            bad[row, head, column] = (math.nan, math.inf, -math.inf)[n % 3]
            fine[row:int(end[row]), head * ratio:(head + 1) * ratio, column] = False
        for _ in range(2):
            got = pkg.attention.packed_attention(q, k, bad, offsets)
            assert torch.equal(got[fine], clean[fine]) and not bool(got[~fine].isfinite().any())
        assert torch.equal(pkg.attention.packed_attention(q, k, v, offsets), clean)
    assert pkg.linear.kernel_status() == 0
