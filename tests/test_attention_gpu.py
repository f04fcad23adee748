"""Cross attention and the int8 cache (gpu_cross_attention, gpu_kv8_append, gpu_kv8_dequant, gpu_kv8_attention) against their formulas in
64 bits.

What an output may be off by, besides half a step of its own type: p is rounded to the products' type (half a step u of each term; fp16 for
the int8 cache; below fp16's normal numbers 2^-25 of the largest p), logits are f32 sums of D products (2^-23 of their absolute terms for
each, and 2^-22 of the logit for its scaling and the exponential's argument), the exponential is good to 2^-21, and the sums over S keys
add 2^-23 of their terms each. With a = sum p |v| / sum p all of it is relative to a; p and the sum of p each carry the logits' error."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _reference(q, k, v, seen, scale):
    """One head: q [L, D], k, v [S, D] in 64 bits (what is not seen may hold anything), seen [L, S] -> (out, bound without the output's rounding
    per unit of u)."""
    L, D = q.shape
    S = k.shape[0]
    if S == 0:
        return torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    some = seen.any(0)
    k, v = torch.where(some[:, None], k, 0.0), torch.where(some[:, None], v, 0.0)
    z = torch.where(seen, q @ k.t() * scale, -math.inf)
    top = z.amax(1, keepdim=True).nan_to_num(neginf=0.0)
    p = torch.exp(z - top)
    mass = p.sum(1, keepdim=True)
    mass1 = torch.where(mass > 0, mass, 1.0)
    a = p @ v.abs() / mass1
    terms = torch.where(seen, q.abs() @ k.abs().t() * abs(scale), 0.0).amax(1, keepdim=True)
    logits = torch.where(seen, z.abs(), 0.0).amax(1, keepdim=True)
    rel = 2 * (D * 2.0 ** -23 * terms + 2.0 ** -22 * logits * 2 + 2.0 ** -21) + 2 * S * 2.0 ** -23
    return p @ v / mass1, a, rel * a + S * 2.0 ** -24 * v.abs().amax() * (mass > 0)


def _check(got, want, a, rest, u):
    half = torch.finfo(got.dtype).eps / 2
    bound = half * want.abs() + (1 + half) * (u * a + rest) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-37)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), ((err / bound.clamp_min(1e-300)).max().item(), err.max().item())


# ---- cross attention ---------------------------------------------------------------------------------------------------------------

def _cross_check(got, q, k, v, seen, scale):
    B, L, H, D = q.shape
    ratio = H // k.shape[2]
    for b in range(B):
        for h in range(H):
            want, a, rest = _reference(q[b, :, h].double(), k[b, :, h // ratio].double(), v[b, :, h // ratio].double(), seen[b][None].expand(L, -1), scale)
            _check(got[b, :, h], want, a, rest, torch.finfo(q.dtype).eps / 2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lkv,H,Hkv,D", [(1, 1, 1, 1, 1, 8), (2, 64, 77, 2, 2, 64), (1, 65, 64, 3, 1, 40), (2, 100, 154, 4, 2, 80), (1, 333, 333, 2, 2, 128),
                                              (3, 7, 65, 6, 2, 160), (1, 130, 512, 1, 1, 256), (1, 5, 2048, 2, 1, 64), (1, 1, 1500, 1, 1, 200), (2, 129, 63, 5, 5, 96),
                                              (1, 1000, 257, 2, 1, 128), (1, 384, 128, 8, 8, 64), (2, 257, 129, 3, 3, 128),
                                              # two tiles of 128 rows a CTA: one and several key tiles, ragged rows, half a tile, shared heads, more items than SMs
                                              (2, 300, 77, 8, 8, 64), (1, 1000, 257, 4, 2, 128), (3, 129, 513, 8, 4, 40), (1, 4096, 130, 1, 1, 80), (2, 2500, 1, 16, 16, 16), (1, 9800, 384, 5, 5, 128)])
def test_cross_attention(pkg, dev, B, Lq, Lkv, H, Hkv, D, dtype):
    g = torch.Generator().manual_seed(B + Lq * 3 + Lkv + D)
    dt = DT[dtype]
    q, k, v = (torch.randn(B, n, h, D, generator=g).mul(s).to(dt).to(dev) for n, h, s in ((Lq, H, 2.0), (Lkv, Hkv, 1.5), (Lkv, Hkv, 1.0)))
    every = torch.ones(B, Lkv, dtype=torch.bool, device=dev)
    _cross_check(pkg.attention.cross_attention(q, k, v), q, k, v, every, D ** -0.5)
    kv_len = torch.randint(0, Lkv + 1, (B,), generator=g, dtype=torch.int32).to(dev)
    mask = (torch.rand(B, Lkv, generator=g) < 0.7).to(dev)
    if B > 1:
        kv_len[1] = 0                                # a sequence without keys
        mask[0] = False                              # and one whose mask leaves none
    under = torch.arange(Lkv, device=dev) < kv_len[:, None]
    for kw, seen in (({"kv_len": kv_len}, under), ({"key_mask": mask}, mask), ({"kv_len": kv_len, "key_mask": mask, "scale": 0.3}, under & mask)):
        # what is not seen holds what it likes
        k1, v1 = (torch.where(seen[:, :, None, None], t, torch.tensor(float("nan"), dtype=dt, device=dev)) for t in (k, v))
        out = torch.full((B, Lq + 1, H, D), 9.0, dtype=dt, device=dev)
        got = pkg.attention.cross_attention(q, k1, v1, out=out[:, :Lq], **kw)
        _cross_check(got, q, k1.nan_to_num(0.0), v1.nan_to_num(0.0), seen, kw.get("scale", D ** -0.5))
        assert bool((out[:, Lq] == 9.0).all())
        if B > 1 and "kv_len" in kw:
            assert bool((got[1] == 0).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lkv,H,D", [(4, 1100, 77, 40, 64), (8, 300, 128, 40, 128), (16, 128, 33, 30, 80), (15, 385, 130, 16, 64)])
def test_cross_attention_with_several_items_to_a_cta(pkg, dev, B, Lq, Lkv, H, D, dtype):
    """Three items and more to each SM's CTA, among them items without a second tile of 128 rows, over one key tile and over two."""
    g = torch.Generator().manual_seed(B + Lq)
    q, k, v = (torch.randn(B, n, H, D, generator=g).to(DT[dtype]).to(dev) for n in (Lq, Lkv, Lkv))
    assert -(-Lq // 256) * B * H > 3 * torch.cuda.get_device_properties(dev).multi_processor_count
    kv_len = torch.randint(1, Lkv + 1, (B,), generator=g, dtype=torch.int32)
    kv_len[1] = 0
    kv_len = kv_len.to(dev)
    for kw, seen in (({}, torch.ones(B, Lkv, dtype=torch.bool, device=dev)), ({"kv_len": kv_len}, torch.arange(Lkv, device=dev) < kv_len[:, None])):
        got = pkg.attention.cross_attention(q, k, v, **kw)
        _cross_check(got, q, k, v, seen, D ** -0.5)
        assert all(torch.equal(pkg.attention.cross_attention(q, k, v, **kw), got) for _ in range(3))
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("Lq", [3, 300])
def test_strides_of_fused_projections(pkg, dev, Lq):
    """q, k and v as slices of wider projections, the result into one, heads before rows, one k and v for the whole batch."""
    g = torch.Generator().manual_seed(Lq)
    B, H, D, Lkv = 2, 3, 64, 90
    every = torch.ones(B, Lkv, dtype=torch.bool, device=dev)
    qkv = torch.randn(B, Lq, 3 * H * D, generator=g).half().to(dev)
    kv = torch.randn(B, Lkv, 2, H, D, generator=g).half().to(dev)
    q = qkv[:, :, H * D:2 * H * D].unflatten(2, (H, D))
    wide = torch.full((B, Lq, 2, H, D), 3.0, dtype=torch.float16, device=dev)
    pkg.attention.cross_attention(q, kv[:, :, 0], kv[:, :, 1], out=wide[:, :, 1])
    _cross_check(wide[:, :, 1], q, kv[:, :, 0], kv[:, :, 1], every, D ** -0.5)
    assert bool((wide[:, :, 0] == 3.0).all())
    t = torch.randn(B, H, Lq, D, generator=g).half().to(dev).transpose(1, 2)
    one = kv[:1].expand(B, Lkv, 2, H, D)
    got = pkg.attention.cross_attention(t, one[:, :, 0], one[:, :, 1], out=torch.empty_like(t))
    _cross_check(got, t, one[:, :, 0], one[:, :, 1], every, D ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_steep_rows(pkg, dev, dtype):
    """Logits of some hundreds, the largest first, last, or in the middle: nothing overflows, the sums follow the largest."""
    g = torch.Generator().manual_seed(0)
    D, Lkv = 64, 300
    q = torch.full((1, 70, 1, D), 4.0).to(DT[dtype]).to(dev)
    v = torch.randn(1, Lkv, 1, D, generator=g).to(DT[dtype]).to(dev)
    every = torch.ones(1, Lkv, dtype=torch.bool, device=dev)
    for order in (torch.arange(Lkv), torch.arange(Lkv).flip(0), torch.randperm(Lkv, generator=g)):
        k = ((order.float()[None, :, None, None] - 150) * 0.1).expand(1, Lkv, 1, D).contiguous().to(DT[dtype]).to(dev)
        _cross_check(pkg.attention.cross_attention(q, k, v), q, k, v, every, D ** -0.5)
        _cross_check(pkg.attention.cross_attention(q, k, v, scale=-D ** -0.5), q, k, v, every, -D ** -0.5)


@pytest.mark.parametrize("M_pixels", [64, 1000])
def test_unet_cross_attention_half(pkg, dev, M_pixels):
    """The run that the operator is for: layer norm and quantizer, q projection, attention to the prompt's projected states, quantizer, output
    projection onto the residual, through the library's own calls; the attention's part against 64 bits on what the projections gave."""
    L, A = pkg.linear, pkg.attention
    g = torch.Generator().manual_seed(M_pixels)
    C, H, ctx, Lkv, images = 640, 10, 768, 77, 2
    M = images * M_pixels

    def weight(n, k, rot):
        q, s = L.sd_quant_rows((torch.randn(n, k, generator=g) * 0.05).half().to(dev), rot)
        return q, s, (torch.randn(n, generator=g) * 0.01).half().to(dev)
    t = torch.randn(M, C, generator=g).half().to(dev)
    states = torch.randn(images * Lkv, ctx, generator=g).half().to(dev)
    wq, wk, wv, wo = weight(C, C, 64), weight(C, ctx, 256), weight(C, ctx, 256), weight(C, C, 64)
    a, xs = L.sd_ln_quant_rows(t, torch.ones(C, device=dev), torch.zeros(C, device=dev), 1e-5, 64)
    q = L.int8_gemm(a, wq[0], xs, wq[1], wq[2], out_dtype=torch.float16).view(images, M_pixels, H, C // H)
    a, xs = L.sd_quant_rows(states, 256)
    k, v = (L.int8_gemm(a, w[0], xs, w[1], w[2], out_dtype=torch.float16).view(images, Lkv, H, C // H) for w in (wk, wv))
    kv_len = torch.tensor([77, 12], dtype=torch.int32, device=dev)
    y = A.cross_attention(q, k, v, kv_len=kv_len)
    _cross_check(y, q, k, v, torch.arange(Lkv, device=dev) < kv_len[:, None], (C // H) ** -0.5)
    ones = torch.ones(C, dtype=torch.float16, device=dev)
    out = L.int8_gemm(*_codes(L, y.view(M, C), wo), wo[2], rscale=ones, resid=t, out=torch.empty_like(t))
    assert out.shape == t.shape and bool(torch.isfinite(out).all()) and L.kernel_status() == 0


def _codes(L, rows, w):
    a, xs = L.sd_quant_rows(rows, 64)
    return a, w[0], xs, w[1]


# ---- the cache -----------------------------------------------------------------------------------------------------------------------

def _cache(pkg, dev, g, B, lens, Hkv, D, T, extra=2):
    width = max(max(lens), 1) // T + extra
    pages = B * width + 3
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32).to(dev)
    c = pkg.attention.Kv8Cache.empty(pages, Hkv, D, T, dev)
    c.k.copy_(torch.randint(-127, 128, c.k.shape, generator=g, dtype=torch.int32).to(torch.int8))
    c.v.copy_(torch.randint(-127, 128, c.v.shape, generator=g, dtype=torch.int32).to(torch.int8))
    c.k_scale.copy_(torch.rand(pages, Hkv, generator=g) * 0.03 + 0.005)
    c.v_scale.copy_(torch.rand(pages, Hkv, generator=g) * 0.03 + 0.005)
    return c, table


def _rows(codes, scale, table, b, n, h):
    T = codes.shape[2]
    page = table[b, :-(-n // T)].long()
    return (codes[page, h].double() * scale[page, h].double()[:, None, None]).flatten(0, 1)[:n]


def _kv8_check(got, q, c, table, lens, q_lens, causal, scale):
    B, L, H, D = q.shape
    ratio = H // c.k.shape[1]
    for b in range(B):
        n, a = lens[b], q_lens[b]
        at = torch.arange(n - a, n, device=q.device)[:, None]
        t = torch.arange(n, device=q.device)[None]
        seen = (t <= at) if causal else torch.ones(a, n, dtype=torch.bool, device=q.device)
        for h in range(H):
            k, v = _rows(c.k, c.k_scale, table, b, n, h // ratio), _rows(c.v, c.v_scale, table, b, n, h // ratio)
            want, mass, rest = _reference(q[b, :a, h].double(), k, v, seen, scale)
            _check(got[b, :a, h], want, mass, rest, 2.0 ** -11)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("B,L,lens,H,Hkv,D,T", [(1, 1, [1], 1, 1, 64, 16), (1, 1, [1999], 32, 8, 128, 64), (3, 1, [0, 1, 700], 8, 8, 64, 64), (2, 1, [65, 4097], 8, 1, 96, 32),
                                                (2, 3, [3, 200], 6, 2, 80, 16), (1, 70, [333], 4, 2, 128, 128), (2, 130, [130, 1000], 3, 1, 64, 32), (1, 16, [2000], 16, 1, 256, 128),
                                                (2, 5, [2, 40], 2, 2, 256, 64), (1, 300, [300], 4, 4, 160, 64), (4, 2, [127, 128, 129, 2], 4, 4, 16, 16), (1, 1, [9000], 4, 4, 128, 64),
                                                (1, 257, [700], 2, 2, 128, 64), (5, 1, [1, 64, 65, 1023, 5000], 24, 2, 64, 16), (1, 9, [1500], 14, 2, 112, 32), (33, 1, list(range(33)), 2, 1, 64, 16),
                                                # two tiles of 128 rows a CTA
                                                (2, 300, [300, 700], 16, 16, 128, 64), (1, 260, [1000], 64, 16, 64, 16), (3, 140, [140, 333, 150], 24, 8, 96, 32), (2, 1000, [1000, 1], 12, 12, 80, 128),
                                                (34, 130, [130 + 7 * i for i in range(34)], 2, 2, 128, 16), (1, 2600, [2600], 8, 8, 128, 32)])
def test_kv8_attention(pkg, dev, B, L, lens, H, Hkv, D, T, dtype):
    g = torch.Generator().manual_seed(B + L + sum(lens) + D)
    c, table = _cache(pkg, dev, g, B, lens, Hkv, D, T)
    q = (torch.randn(B, L, H, D, generator=g) * 1.5).to(DT[dtype]).to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = pkg.attention.kv8_attention(q, c, table, n, causal=False)
    _kv8_check(got, q, c, table, lens, [L] * B, False, D ** -0.5)
    q_lens = [min(L, m) for m in lens]
    out = torch.full((B, L + 1, H, D), 9.0, dtype=DT[dtype], device=dev)
    got = pkg.attention.kv8_attention(q, c, table, n, q_len=torch.tensor(q_lens, dtype=torch.int32, device=dev), scale=0.2, out=out[:, :L])
    _kv8_check(got, q, c, table, lens, q_lens, True, 0.2)
    for b in range(B):
        assert bool((out[b, q_lens[b]:] == 9.0).all())
    got = pkg.attention.kv8_attention(q, c, table, n)      # rows before the sequence's first token see nothing
    for b in range(B):
        assert bool((got[b, :max(0, L - lens[b])] == 0).all())
    _kv8_check(got[:, L - min(q_lens):], q[:, L - min(q_lens):], c, table, lens, [min(q_lens)] * B, True, D ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("B,L,ratio,Hkv,D,T", [(20, 300, 1, 24, 64, 16), (23, 64, 2, 20, 128, 32), (40, 65, 2, 12, 96, 64), (12, 385, 1, 20, 16, 128)])
def test_kv8_attention_with_several_items_to_a_cta(pkg, dev, B, L, ratio, Hkv, D, T, dtype):
    """Three items and more to each SM's CTA, of one row tile, of two, and of both in turn: what one item leaves is not taken for the next one's."""
    g = torch.Generator().manual_seed(B + L)
    lens = [L + (37 * b) % 200 for b in range(B)]
    lens[3] = 0
    c, table = _cache(pkg, dev, g, B, lens, Hkv, D, T)
    q = (torch.randn(B, L, Hkv * ratio, D, generator=g) * 1.5).to(DT[dtype]).to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    assert -(-L * ratio // 256) * B * Hkv > 3 * torch.cuda.get_device_properties(dev).multi_processor_count
    for causal in (True, False):
        got = pkg.attention.kv8_attention(q, c, table, n, causal=causal)
        _kv8_check(got, q, c, table, lens, [min(L, m) for m in lens], causal, D ** -0.5)
        assert bool((got[3] == 0).all()) and all(torch.equal(pkg.attention.kv8_attention(q, c, table, n, causal=causal), got) for _ in range(3))
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("size", [1e-20, 1e-4, 1.0, 3e4, 1e20])
def test_bf16_queries_of_any_size(pkg, dev, size):
    """A row of queries is taken times a power of two: large and small ones are as good as others."""
    g = torch.Generator().manual_seed(7)
    c, table = _cache(pkg, dev, g, 1, [200], 2, 64, 32)
    q = (torch.randn(1, 3, 4, 64, generator=g) * size).bfloat16().to(dev)
    n = torch.tensor([200], dtype=torch.int32, device=dev)
    got = pkg.attention.kv8_attention(q, c, table, n, scale=0.1 / size)
    _kv8_check(got, q, c, table, [200], [3], True, 0.1 / size)


@pytest.mark.parametrize("L,H,lens", [(3, 4, [200]), (300, 16, [300, 333, 400, 310])])
@pytest.mark.parametrize("power", [118, 128, -100, -122, -131])
def test_bf16_queries_at_the_ends_of_the_range(pkg, dev, L, H, lens, power):
    """Rows up to the type's largest numbers and down to its subnormal ones, by few rows and by many. Logits of some units, and of some
    thousands for the largest: scale * k_scale is kept to f32's normal numbers."""
    g = torch.Generator().manual_seed(power + 200)
    B, Hkv, D, T = len(lens), 2 if L < 100 else 16, 64, 32
    c, table = _cache(pkg, dev, g, B, lens, Hkv, D, T)
    shift = -8 if power > 0 else 6
    c.k_scale.mul_(2.0 ** shift)
    q = torch.randn(B, L, H, D, generator=g).clamp(-3.9, 3.9).mul(2.0 ** (power - 2)).bfloat16().to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    scale = 2.0 ** (max(-power, -118) - shift)
    assert bool(torch.isfinite(q).all()) and float(q.float().abs().max()) > 2.0 ** (power - 1)
    got = pkg.attention.kv8_attention(q, c, table, n, scale=scale)
    _kv8_check(got, q, c, table, lens, [L] * B, True, scale)


def test_scales_far_apart(pkg, dev):
    """Pages whose values differ by many orders of magnitude: p carries the value's scale, so the largest contribution keeps fp16's bits
    whatever the others' size; a page of zeros (scale 1e-30, or 0 where nothing was ever written) only weighs in the sum of p."""
    g = torch.Generator().manual_seed(8)
    D, T, n = 64, 16, 16 * 12
    for dt in ("f16", "bf16"):
        c, table = _cache(pkg, dev, g, 1, [n], 1, D, T)
        page = table[0].long()
        for j, s in enumerate((1e-6, 1.0, 1e-30, 1e-3, 1e3, 1e-12)):
            c.v_scale[page[2 * j]] = s
        c.v[page[4]] = 0
        c.v[page[5]], c.v_scale[page[5]] = 0, 0.0
        q = (torch.randn(1, 2, 2, D, generator=g)).to(DT[dt]).to(dev)
        length = torch.tensor([n], dtype=torch.int32, device=dev)
        _kv8_check(pkg.attention.kv8_attention(q, c, table, length), q, c, table, [n], [2], True, D ** -0.5)
        for keep in (4, 5):          # every other page far below: mostly the page of zeros is seen
            c.k_scale[page] = 0.0
            c.k_scale[page[keep]] = 0.2
            _kv8_check(pkg.attention.kv8_attention(q, c, table, length), q, c, table, [n], [2], True, D ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("L,H,Hkv,lens", [(40, 2, 2, [100, 90]), (300, 16, 16, [400, 350, 300, 310, 320, 330])])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_a_scale_that_is_no_number(pkg, dev, L, H, Hkv, lens, dtype, which):
    """A page whose scale of K or of V is NaN: rows that see one of its keys are NaN, as what it stands for is; rows before it are not touched."""
    g = torch.Generator().manual_seed(L)
    B, D, T = len(lens), 64, 16
    c, table = _cache(pkg, dev, g, B, lens, Hkv, D, T)
    q = torch.randn(B, L, H, D, generator=g).to(DT[dtype]).to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    want = pkg.attention.kv8_attention(q, c, table, n)
    slot = (lens[1] - 20) // T
    getattr(c, which)[table[1, slot].long(), 0] = float("nan")
    got = pkg.attention.kv8_attention(q, c, table, n)
    sees = torch.arange(lens[1] - L, lens[1], device=dev) >= slot * T
    hit = torch.zeros(B, L, H, dtype=torch.bool, device=dev)
    hit[1, sees, :H // Hkv] = True
    assert 0 < int(sees.sum()) < L
    assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], want[~hit])


def test_what_is_never_seen_may_hold_anything(pkg, dev):
    """Behind a sequence's last token: codes and scales of unused pages (NaN), table entries that are no pages at all."""
    g = torch.Generator().manual_seed(9)
    lens = [0, 17, 100]
    c, table = _cache(pkg, dev, g, 3, lens, 2, 64, 32, extra=4)
    used = torch.cat([table[b, :-(-n // 32)] for b, n in enumerate(lens)]).long()
    unused = torch.ones(c.k.shape[0], dtype=torch.bool, device=dev)
    unused[used] = False
    c.k_scale[unused], c.v_scale[unused] = float("nan"), float("inf")
    for b, n in enumerate(lens):
        table[b, -(-n // 32):] = torch.tensor([2 ** 31 - 1, -1, -2 ** 31], dtype=torch.int32, device=dev).repeat(4)[:table.shape[1] - -(-n // 32)]
    q = torch.randn(3, 2, 4, 64, generator=g).half().to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    q_lens = [0, 2, 2]
    got = pkg.attention.kv8_attention(q, c, table, n, q_len=torch.tensor(q_lens, dtype=torch.int32, device=dev))
    _kv8_check(got, q, c, table, lens, q_lens, True, 64 ** -0.5)
    assert bool((got[0] == 0).all())
    k, v = pkg.attention.kv8_dequant(c, table, n, 130)
    for b, m in enumerate(lens):
        assert bool((k[b, m:] == 0).all()) and bool((v[b, m:] == 0).all())
        for h in range(2):
            assert torch.equal(k[b, :m, h], _rows(c.k, c.k_scale, table, b, m, h).float()) and torch.equal(v[b, :m, h], _rows(c.v, c.v_scale, table, b, m, h).float())
    # a page in the middle that does not exist: its tokens are not seen; lengths beyond the table end with it
    table[2, 1] = -5
    t = torch.arange(100, device=dev)
    seen = ((t < 32) | (t >= 64))[None].expand(2, 100) & (t[None] <= torch.tensor([[98], [99]], device=dev))
    got = pkg.attention.kv8_attention(q, c, table, n)
    real = table.clone()
    real[2, 1] = used[0]
    for h in range(4):
        want, a, rest = _reference(q[2, :, h].double(), _rows(c.k, c.k_scale, real, 2, 100, h // 2), _rows(c.v, c.v_scale, real, 2, 100, h // 2), seen, 64 ** -0.5)
        _check(got[2, :, h], want, a, rest, 2.0 ** -11)


def _append_as_defined(codes, scale, table, start, count, rows):
    """Page by page in f32; divisions and roundings are those of the definition, one each."""
    codes, scale = codes.clone(), scale.clone()
    T, (W, pages) = codes.shape[2], (table.shape[1], codes.shape[0])
    for b in range(rows.shape[0]):
        s0, n = int(start[b]), min(int(count[b]), rows.shape[1])
        if s0 < 0 or n <= 0:
            continue
        for slot in range(s0 // T, (s0 + n - 1) // T + 1):
            lo, hi = max(s0, slot * T), min(s0 + n, (slot + 1) * T)
            if slot >= W or not 0 <= int(table[b, slot]) < pages:
                continue
            page, at = int(table[b, slot]), lo - slot * T
            new = rows[b, lo - s0:hi - s0].float().transpose(0, 1)           # [Hkv, n, D]
            top = new.abs().nan_to_num(0.0).amax((1, 2)).clamp_max(torch.finfo(torch.float32).max)
            s = (top * (1 / 127)).clamp_min(1e-30)
            if at > 0:
                s = torch.maximum(s, scale[page])
                codes[page, :, :at] = torch.round(codes[page, :, :at].float() * (scale[page] / s)[:, None, None]).to(torch.int8)
            codes[page, :, at:at + hi - lo] = torch.round(new / s[:, None, None]).nan_to_num(0.0).clamp(-127, 127).to(torch.int8)
            scale[page] = s
    return codes, scale


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("L,start,count,Hkv,D,T", [(1, [0, 15, 16, 700], [1, 1, 1, 1], 8, 128, 64), (5, [14, 0, 31], [5, 0, 3], 2, 64, 16), (200, [0, 3, 129], [200, 77, 1], 3, 80, 32),
                                                   (1000, [24], [1000], 1, 256, 128), (33, [31, -4, 32], [40, 5, -2], 4, 16, 32)])
def test_append(pkg, dev, L, start, count, Hkv, D, T, dtype):
    g = torch.Generator().manual_seed(L + D)
    B = len(start)
    c, table = _cache(pkg, dev, g, B, [max(s + n for s, n in zip(start, count))], Hkv, D, T)
    table = table[:1] if B == 1 else torch.randperm(c.k.shape[0], generator=g)[:c.k.shape[0] // B * B].view(B, -1).to(torch.int32).to(dev)
    size = torch.tensor([0.05, 1.0, 30.0]).repeat(B)[:B, None, None, None]      # both sides of the scales that the pages have
    k, v = (torch.randn(B, L, Hkv, D, generator=g).mul(size).to(DT[dtype]).to(dev) for _ in range(2))
    s, n = torch.tensor(start, dtype=torch.int32, device=dev), torch.tensor(count, dtype=torch.int32, device=dev)
    want_k = _append_as_defined(c.k, c.k_scale, table, start, count, k)
    want_v = _append_as_defined(c.v, c.v_scale, table, start, count, v)
    pkg.attention.kv8_append(c, k, v, table, s, n)
    assert torch.equal(c.k, want_k[0]) and torch.equal(c.k_scale, want_k[1]) and torch.equal(c.v, want_v[0]) and torch.equal(c.v_scale, want_v[1])
    pkg.attention.kv8_append(c, k, v, table, s, n)      # the same rows again change nothing
    assert torch.equal(c.k, want_k[0]) and torch.equal(c.k_scale, want_k[1])


def test_append_edges(pkg, dev):
    """Infinities, NaN, rows of zeros, strided rows, pages and places outside the cache."""
    g = torch.Generator().manual_seed(12)
    c, table = _cache(pkg, dev, g, 2, [100], 2, 64, 32)
    k = torch.randn(2, 40, 2, 64, generator=g).to(dev)
    k[0, 3, 0, 5], k[0, 4, 1, 6], k[1, :, 0] = float("inf"), float("nan"), 0.0
    wide = torch.randn(2, 40, 3, 2, 64, generator=g).to(dev)
    wide[:, :, 1] = k
    table[1, 1] = -1
    start, count = [0, 10], [40, 40]
    s, n = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (start, count))
    want_k, want_v = _append_as_defined(c.k, c.k_scale, table, start, count, k), _append_as_defined(c.v, c.v_scale, table, start, count, wide[:, :, 2])
    pkg.attention.kv8_append(c, wide[:, :, 1], wide[:, :, 2], table, s, n)
    assert torch.equal(c.k, want_k[0]) and torch.equal(c.k_scale, want_k[1]) and torch.equal(c.v, want_v[0]) and torch.equal(c.v_scale, want_v[1])
    before = c.k.clone()
    pkg.attention.kv8_append(c, k, k, table, torch.tensor([10 ** 9, 2 ** 31 - 3], dtype=torch.int32, device=dev))      # behind every page
    assert torch.equal(c.k, before)


def test_a_sequence_grows_token_by_token(pkg, dev):
    """A prompt, then single tokens: each value is off by half a step of its page's scale, and half a step more for each time that the scale
    of its page was raised; attention after every step against 64 bits on what the cache holds."""
    A = pkg.attention
    g = torch.Generator().manual_seed(4)
    B, H, Hkv, D, T = 2, 4, 2, 64, 16
    c = A.Kv8Cache.empty(20, Hkv, D, T, dev)
    table = torch.randperm(20, generator=g)[:12].view(B, 6).to(torch.int32).to(dev)
    k, v = (torch.randn(B, 60, Hkv, D, generator=g).bfloat16().to(dev) for _ in range(2))
    prompt = [21, 5]
    lens = torch.tensor(prompt, dtype=torch.int32, device=dev)
    A.kv8_append(c, k[:, :21], v[:, :21], table, torch.zeros_like(lens), lens)
    for i in range(20):
        at = lens.tolist()
        one = torch.stack([k[b, at[b]] for b in range(B)])[:, None], torch.stack([v[b, at[b]] for b in range(B)])[:, None]
        A.kv8_append(c, *one, table, lens)
        lens = lens + 1
        q = torch.randn(B, 1, H, D, generator=g).bfloat16().to(dev)
        _kv8_check(A.kv8_attention(q, c, table, lens), q, c, table, lens.tolist(), [1, 1], True, D ** -0.5)
    for b, n in enumerate(lens.tolist()):
        back, _ = A.kv8_dequant(c, table, lens, n)
        step = c.k_scale[table[b].long()].repeat_interleave(T, 0)[:n, :, None].double()
        assert bool(((back[b].double() - k[b, :n].double()).abs() <= step * (0.5 + 0.5 * T + 1e-4)).all())


def test_replayed_from_a_graph_with_longer_sequences(pkg, dev):
    """A captured step reads lengths from the device: replayed it serves the sequence as it has grown. Nothing but the caller's buffers is used."""
    A = pkg.attention
    g = torch.Generator().manual_seed(6)
    B, H, Hkv, D, T = 2, 8, 2, 128, 64
    c, table = _cache(pkg, dev, g, B, [3000], Hkv, D, T)
    q = torch.randn(B, 1, H, D, generator=g).half().to(dev)
    kv = torch.randn(B, 1, Hkv, D, generator=g).half().to(dev)
    lens = torch.tensor([10, 2000], dtype=torch.int32, device=dev)
    out, side = torch.empty_like(q), torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        def step():
            A.kv8_append(c, kv, kv, table, lens)
            lens.add_(1)
            A.kv8_attention(q, c, table, lens, out=out)
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for _ in range(3):
            graph.replay()
        side.synchronize()
    assert lens.tolist() == [14, 2004]
    _kv8_check(out, q, c, table, lens.tolist(), [1, 1], True, D ** -0.5)
    assert all(torch.equal(A.kv8_attention(q, c, table, lens), out) for _ in range(3))


def test_pages_beyond_32_bits(pkg, dev):
    """A cache of more than 2^31 bytes of keys, with sequences on its last pages: written, read back, attended to by few rows and by many."""
    A = pkg.attention
    g = torch.Generator().manual_seed(13)
    pages, Hkv, D, T = 17000, 8, 128, 128
    c = A.Kv8Cache.empty(pages, Hkv, D, T, dev)
    table = torch.tensor([[pages - 1, 0, pages - 2], [pages - 5, pages - 3, 1]], dtype=torch.int32, device=dev)
    k, v = (torch.randn(2, 300, Hkv, D, generator=g).half().to(dev) for _ in range(2))
    start = torch.zeros(2, dtype=torch.int32, device=dev)
    n = torch.tensor([300, 290], dtype=torch.int32, device=dev)
    A.kv8_append(c, k, v, table, start, n)
    back, _ = A.kv8_dequant(c, table, n, 300)
    for b, m in enumerate(n.tolist()):
        step = c.k_scale[table[b].long()].repeat_interleave(T, 0)[:m, :, None]
        assert bool(((back[b, :m] - k[b, :m].float()).abs() <= step * 0.5001).all())
    for L, H in ((1, 32), (200, 16), (260, 32)):
        q = torch.randn(2, L, H, D, generator=g).half().to(dev)
        _kv8_check(A.kv8_attention(q, c, table, n), q, c, table, [300, 290], [L, L], True, D ** -0.5)


@pytest.mark.parametrize("Lq,Lkv,H", [(128, 2 ** 26, 64), (128, 2 ** 26 + 77, 64), (2, 2 ** 25 + 5, 8)])
def test_very_many_keys(pkg, dev, Lq, Lkv, H):
    """A few keys spread over the whole length have logits of about 60, all others 0: together less than 2^27 e^-60 = 1.2e-18 of the sums, so that the rows
    are those of the few keys alone."""
    g = torch.Generator().manual_seed(Lq + Lkv)
    D = 64
    k, v = (torch.zeros(1, Lkv, 1, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    at = torch.tensor([0, 1, 127, 128, Lkv // 3, Lkv // 2, 2 ** 23 + 1, Lkv - 129, Lkv - 1], device=dev)
    k[0, at, 0] = (1 + 0.05 * torch.randn(len(at), D, generator=g)).bfloat16().to(dev)
    v[0, at, 0] = torch.randn(len(at), D, generator=g).bfloat16().to(dev)
    q = (7.5 + 0.1 * torch.randn(1, Lq, H, D, generator=g)).bfloat16().to(dev)
    got = pkg.attention.cross_attention(q, k, v)
    few = torch.ones(1, len(at), dtype=torch.bool, device=dev)
    _cross_check(got, q, k[:, at], v[:, at], few, D ** -0.5)
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("Lq,Hkv,pages", [(1, 8, 2 ** 14), (256, 96, 2 ** 11)])
def test_very_many_tokens_of_the_cache(pkg, dev, Lq, Hkv, pages):
    """The same over the cache: two million tokens for single rows, a quarter of a million for many."""
    g = torch.Generator().manual_seed(pages)
    D, T = 64, 128
    n = pages * T - 5
    c = pkg.attention.Kv8Cache.empty(pages, Hkv, D, T, dev)
    c.k_scale.fill_(0.01), c.v_scale.fill_(0.02)
    table = torch.randperm(pages, generator=g).to(torch.int32).to(dev)[None]
    at = torch.tensor([0, 1, 127, 128, n // 3, n // 2, n - 300, n - 257], device=dev)
    page, row = table[0, at // T].long(), at % T
    k8 = torch.randint(90, 110, (len(at), Hkv, D), generator=g, dtype=torch.int32).to(torch.int8).to(dev)
    v8 = torch.randint(-127, 128, (len(at), Hkv, D), generator=g, dtype=torch.int32).to(torch.int8).to(dev)
    for i in range(len(at)):
        c.k[page[i], :, row[i]], c.v[page[i], :, row[i]] = k8[i], v8[i]
    q = (7.5 + 0.1 * torch.randn(1, Lq, Hkv, D, generator=g)).half().to(dev)
    got = pkg.attention.kv8_attention(q, c, table, torch.tensor([n], dtype=torch.int32, device=dev))
    few = torch.ones(Lq, len(at), dtype=torch.bool, device=dev)
    step = [float(c.k_scale[0, 0]), float(c.v_scale[0, 0])]
    for h in range(Hkv):
        want, a, rest = _reference(q[0, :, h].double(), k8[:, h].double() * step[0], v8[:, h].double() * step[1], few, D ** -0.5)
        _check(got[0, :, h], want, a, rest, 2.0 ** -11)
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("Lq", [1, 40, 600])
def test_two_streams_at_once_and_ordinary_launches(pkg, dev, Lq):
    """Nothing is shared between calls: two at a time give what one gives. Beside a collective's kernels launches are ordinary ones."""
    A, L = pkg.attention, pkg.linear
    g = torch.Generator().manual_seed(Lq)
    c, table = _cache(pkg, dev, g, 2, [900, 700], 8, 64, 32)
    n = torch.tensor([900, 700], dtype=torch.int32, device=dev)
    q = torch.randn(2, Lq, 16, 64, generator=g).half().to(dev)
    kv = torch.randn(2, 150, 8, 64, generator=g).half().to(dev)
    calls = (lambda out: A.kv8_attention(q, c, table, n, out=out), lambda out: A.cross_attention(q, kv, kv, out=out))
    want = [call(torch.zeros_like(q)) for call in calls]
    outs, streams = [torch.zeros_like(q) for _ in range(8)], [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            calls[i // 2 % 2](out)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i // 2 % 2]) for i, out in enumerate(outs))
    was = L.set_gemm_cluster_limit(4)
    try:
        assert all(torch.equal(call(torch.zeros_like(q)), w) for call, w in zip(calls, want))
    finally:
        L.set_gemm_cluster_limit(was)
    assert L.kernel_status() == 0


@pytest.mark.parametrize("Lq", [2, 300])
def test_pages_shared_by_sequences(pkg, dev, Lq):
    """Two sequences with the same first pages (a prefix), and one with a page twice: attention only reads them."""
    g = torch.Generator().manual_seed(Lq)
    c, table = _cache(pkg, dev, g, 3, [400], 12, 64, 32)
    table[1, :5], table[2, 3] = table[0, :5], table[2, 0]
    q = torch.randn(3, Lq, 24, 64, generator=g).bfloat16().to(dev)
    lens = [400, 390, 333]
    _kv8_check(pkg.attention.kv8_attention(q, c, table, torch.tensor(lens, dtype=torch.int32, device=dev)), q, c, table, lens, [Lq] * 3, True, 64 ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Lq", [1, 70, 700])
def test_in_place_of_the_queries(pkg, dev, Lq, dtype):
    A = pkg.attention
    g = torch.Generator().manual_seed(Lq)
    B, H, Hkv, D = 2, 24, 8, 64
    c, table = _cache(pkg, dev, g, B, [1500, 900], Hkv, D, 32)
    n = torch.tensor([1500, 900], dtype=torch.int32, device=dev)
    q = torch.randn(B, Lq, H, D, generator=g).to(DT[dtype]).to(dev)
    kv = torch.randn(B, 600, Hkv, D, generator=g).to(DT[dtype]).to(dev)
    for call in (lambda q, out: A.kv8_attention(q, c, table, n, out=out), lambda q, out: A.cross_attention(q, kv, kv, out=out)):
        want = call(q, None)
        for _ in range(3):
            x = q.clone()
            call(x, x)
            assert torch.equal(x, want)


def test_rows_beyond_the_last_and_zero_sizes(pkg, dev):
    """No pages at all, no tokens, a negative length: zeros, or nothing written."""
    A = pkg.attention
    c = A.Kv8Cache.empty(0, 2, 64, 16, dev)
    table, n = torch.zeros(2, 0, dtype=torch.int32, device=dev), torch.tensor([5, -3], dtype=torch.int32, device=dev)
    for Lq in (1, 300):
        q = torch.randn(2, Lq, 32, 64, device=dev).half()
        assert bool((A.kv8_attention(q, c, table, n) == 0).all())
    kv = torch.randn(2, 4, 2, 64, device=dev).half()
    A.kv8_append(c, kv, kv, table, n)
    k, v = A.kv8_dequant(c, table, n, 7, dtype=torch.bfloat16)
    assert k.shape == (2, 7, 2, 64) and bool((k == 0).all()) and bool((v == 0).all())
    assert A.kv8_dequant(c, table, n, 0)[0].shape == (2, 0, 2, 64)


def test_refusals(pkg, dev):
    A = pkg.attention
    q = torch.zeros(2, 3, 4, 64, device=dev).half()
    c = A.Kv8Cache.empty(4, 2, 64, 16, dev)
    t, n = torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    kv = torch.zeros(2, 3, 2, 64, device=dev).half()
    f32 = A.Kv8Cache(c.k.float(), c.v, c.k_scale, c.v_scale)
    for bad in (lambda: A.cross_attention(q, kv, kv[:, :2]), lambda: A.cross_attention(q, kv.float(), kv.float()), lambda: A.cross_attention(q.float(), kv.float(), kv.float()),
                lambda: A.cross_attention(q, kv, kv, kv_len=n.long()), lambda: A.cross_attention(q, kv, kv, key_mask=t.bool()), lambda: A.cross_attention(q[0], kv, kv),
                lambda: A.cross_attention(q[:, :, :3], kv, kv), lambda: A.cross_attention(q, kv, kv.cpu()), lambda: A.cross_attention(q, kv, kv, out=q[:, :2]),
                lambda: A.kv8_attention(q, f32, t, n), lambda: A.kv8_attention(q, c, t.long(), n), lambda: A.kv8_attention(q, c, t[:1], n),
                lambda: A.kv8_attention(q, c, t, n[:1]), lambda: A.kv8_attention(q[..., :32], c, t, n), lambda: A.kv8_attention(q, c, t, n, q_len=n.float()),
                lambda: A.kv8_append(c, q, q, t, n), lambda: A.kv8_append(c, kv, kv.float(), t, n), lambda: A.kv8_append(c, kv, kv, t, n, n.long()),
                lambda: A.kv8_dequant(c, t.long(), n, 4), lambda: A.kv8_dequant(c, t, n[:1], 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(pkg.GpuKernelError, match="-5"):
        A.cross_attention(torch.zeros(2, 3, 4, 65, device=dev).half()[..., 1:], kv, kv)
    with pytest.raises(pkg.GpuKernelError, match="-206"):
        A.kv8_attention(q, A.Kv8Cache.empty(4, 2, 64, 24, dev), t, n)
    assert A.cross_attention(q[:, :0], kv, kv).shape == (2, 0, 4, 64) and bool((A.cross_attention(q, kv[:, :0], kv[:, :0]) == 0).all())
