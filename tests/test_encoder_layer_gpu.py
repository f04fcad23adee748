"""What a text encoder's layer runs between its cache and its weights -- rows normalised into e4m3 (gpu_norm_rows), linears over e4m3 blocks (gpu_f8_*),
rotary positions (gpu_rotary), attention of packed prompts (gpu_packed_attention) -- against the formulas in 64 bits.

Tolerances. A rounding is off by at most half a step of its type (e4m3: 2^-4 of the value, 2^-10 below 2^-6). norm_rows: a row's sum of squares has at
most 80 f32 additions in a chain (2^-24 of the sum each, half of it in the root), the root and its reciprocal 2^-22, three products 2^-24 each: 2^-18
of the value covers them; silu's exponential, sum and quotient stay below 2^-20. f8_linear: products of codes are exact, and an output's additions are off by at
most 2^-23 of the absolute terms for each of K + 4. rotary: the angle keeps 2^-25 of a turn (2^-22.3 radians), sine and cosine 2^-22, products and sums
2^-24 each, the norm 26 x 2^-24: 40 x 2^-24 of |a| + |b|. Attention: as in test_attention_gpu."""
from __future__ import annotations

import math

import pytest
import torch

from test_attention_gpu import _check as _check_attention
from test_attention_gpu import _reference

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn


def _half(t):
    return torch.finfo(t).eps / 2


def _least(t):
    return 2.0 ** -25 if t == torch.float16 else 1e-37


# ---- e4m3 blocks -----------------------------------------------------------------------------------------------------------------

def _blocks(x, rows):
    M, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % 128, 0, -M % rows))
    return x.view(-1, rows, x.shape[1] // 128, 128)


def _formula(x, rows):
    """Codes and scales of x f32 as the library's writers form them, in the same two f32 products."""
    M, K = x.shape
    b = _blocks(x, rows)
    s = b.abs().nan_to_num(0.0, posinf=math.inf).amax((1, 3)).clamp_min(1e-30) * (1.0 / 448.0)
    codes = (b * s.reciprocal()[:, None, :, None]).clamp(-448.0, 448.0).to(F8)
    return codes.reshape(-1, b.shape[2] * 128)[:M, :K].contiguous(), s


def _values(codes, scales, rows):
    s = scales.double().repeat_interleave(rows, 0)[:codes.shape[0]].repeat_interleave(128, 1)[:, :codes.shape[1]]
    return codes.double() * s


def _same_codes(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("N,K", [(1, 16), (5, 128), (127, 144), (128, 128), (129, 1040), (300, 2560), (1000, 48)])
def test_packing(pkg, dev, N, K, dtype):
    g = torch.Generator().manual_seed(N + K)
    w = (torch.randn(N, K, generator=g) * (0.02 + torch.rand(N, 1, generator=g))).to(DT[dtype]).to(dev)
    w[0, 0] = 0.0
    codes, s = pkg.linear.f8_requant(w)
    want, ws = _formula(w.float(), 128)
    assert torch.equal(s, ws) and _same_codes(codes, want)
    wide = torch.full((N, 3 * K), 3.0, dtype=w.dtype, device=dev)
    wide[:, K:2 * K] = w
    if K * w.element_size() % 16 == 0:
        assert _same_codes(pkg.linear.f8_requant(wide[:, K:2 * K])[0], want)
    for out in DT.values():
        back = pkg.linear.f8_dequant(codes, s, dtype=out)
        v = _values(codes, s, 128)
        assert bool(((back.double() - v).abs() <= (_half(out) + 2.0 ** -24) * v.abs() + _least(out)).all())
    rows, rs = pkg.linear.norm_rows(w, pkg.ffi.PRO_PLAIN, out_dtype=F8)
    want, ws = _formula(w.float(), 1)
    assert torch.equal(rs, ws) and _same_codes(rows, want)
    assert torch.equal(pkg.linear.f8_dequant(rows, rs, rows=1), (_values(rows, rs, 1)).float())


def test_blocks_of_zeros_and_numbers_that_are_none(pkg, dev):
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(1)).to(dev)
    x[0] = 0.0
    x[1, 3], x[2, 200] = math.nan, math.inf
    x[3, :128] *= 1e-38
    for codes, s, rows in ((*pkg.linear.norm_rows(x, pkg.ffi.PRO_PLAIN, out_dtype=F8), 1), (*pkg.linear.f8_requant(x[2:3]), 128)):
        want, ws = _formula(x if rows == 1 else x[2:3], rows)
        assert torch.equal(s, ws) and torch.equal(codes.float().isnan(), want.float().isnan()) and torch.equal(codes.float().nan_to_num(0.0), want.float().nan_to_num(0.0))
    codes, s = pkg.linear.norm_rows(x, pkg.ffi.PRO_PLAIN, out_dtype=F8)
    assert bool((codes[0].float() == 0).all()) and bool(s.isfinite()[[0, 1, 3]].all())
    assert int(codes[1].float().isnan().sum()) == 1 and int(codes[2].float().isnan().sum()) == 1


# ---- norm_rows --------------------------------------------------------------------------------------------------------------------

def _check_rows(got, scales, y, rel=2.0 ** -18):
    """got against y in 64 bits: rows of a type, or codes with scales."""
    if scales is None:
        bound = (_half(got.dtype) + rel) * y.abs() + _least(got.dtype)
        assert bool(((got.double() - y).abs() <= bound).all()), ((got.double() - y).abs() / bound).max().item()
        return
    top = _blocks(y, 1).abs().amax((1, 3)).clamp_min(1e-30) / 448.0
    assert bool(((scales.double() - top).abs() <= (rel + 2.0 ** -23) * top).all())
    v = y / scales.double().repeat_interleave(128, 1)[:, :y.shape[1]]
    bound = (2.0 ** -4 * v.abs()).clamp_min(2.0 ** -10) + 2 * rel * v.abs()
    assert bool(((got.double() - v).abs() <= bound).all()), ((got.double() - v).abs() / bound).max().item()


SHAPES = [(1, 16), (1, 2560), (2, 128), (3, 144), (7, 4096), (8, 4112), (5, 9728), (2, 16384), (2, 16400), (1, 32768), (33, 640), (300, 1280), (1000, 256), (600, 2560)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K", SHAPES)
def test_norm_with_the_residual(pkg, dev, M, K, dtype):
    g = torch.Generator().manual_seed(M * 3 + K)
    L, F, dt = pkg.linear, pkg.ffi, DT[dtype]
    x = (torch.randn(M, K, generator=g) * (0.2 + torch.randn(K, generator=g).abs() * 5)).to(dt).to(dev)
    w = (1 + 0.3 * torch.randn(K, generator=g)).to(dev)
    stream = (torch.randn(M, K, generator=g) * 4).to(dt).to(dev)
    sum64 = x.double() + stream.double()
    for out_dt in (F8, dt, torch.float32, torch.bfloat16):
        new = torch.full((M + 1, K), 5.0, dtype=dt, device=dev)
        got = L.norm_rows(x, F.PRO_RMS, norm_w=w, eps=1e-5, resid=stream, resid_out=new[:M], out_dtype=out_dt)
        got, s = got if out_dt == F8 else (got, None)
        assert bool(((new[:M].double() - sum64).abs() <= (_half(dt) + 2.0 ** -24) * sum64.abs() + _least(dt)).all()) and bool((new[M] == 5.0).all())
        n = new[:M].double()
        _check_rows(got, s, n / (n.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double())
    for out_dt in (F8, dt):        # without a stream, without weights; in place of the stream; x's own place
        got = L.norm_rows(x, F.PRO_RMS, eps=1e-6, out_dtype=out_dt)
        got, s = got if out_dt == F8 else (got, None)
        n = x.double()
        _check_rows(got, s, n / (n.square().mean(1, keepdim=True) + 1e-6).sqrt())
    kept, x2 = stream.clone(), x.clone()
    a = L.norm_rows(x, F.PRO_RMS, norm_w=w, eps=1e-5, resid=kept)
    assert torch.equal(kept, new[:M])
    b = L.norm_rows(x2, F.PRO_RMS, norm_w=w, eps=1e-5, resid=stream, resid_out=x2)
    assert torch.equal(x2, kept) and torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K", SHAPES)
def test_swiglu_rows(pkg, dev, M, K, dtype):
    g = torch.Generator().manual_seed(M + K)
    dt = DT[dtype]
    x = (torch.randn(M, 2 * K + 64, generator=g) * 3).to(dt).to(dev)
    a, b = x[:, :K].double(), x[:, K + 16:2 * K + 16].double()
    y = a / (1 + torch.exp(-a)) * b
    for out_dt in (F8, dt):
        got = pkg.linear.norm_rows(x, pkg.ffi.PRO_SWIGLU, K=K, up_offset=K + 16, out_dtype=out_dt)
        got, s = got if out_dt == F8 else (got, None)
        _check_rows(got, s, y, 2.0 ** -20)


def test_norm_rows_in_wider_buffers_and_of_extreme_rows(pkg, dev):
    g = torch.Generator().manual_seed(9)
    L, F = pkg.linear, pkg.ffi
    for dt in DT.values():
        wide = torch.randn(20, 3 * 320, generator=g).to(dt).to(dev)
        out = torch.full((20, 2 * 320), 7.0, dtype=dt, device=dev)
        before = wide.clone()
        L.norm_rows(wide[:, 320:640], F.PRO_RMS, eps=1e-6, resid=wide[:, 640:], out=out[:, 320:])
        s = (before[:, 320:640].float() + before[:, 640:].float()).to(dt)
        assert torch.equal(wide[:, 640:], s) and torch.equal(wide[:, :640], before[:, :640]) and bool((out[:, :320] == 7.0).all())
        n = s.double()
        _check_rows(out[:, 320:], None, n / (n.square().mean(1, keepdim=True) + 1e-6).sqrt())
    x = torch.randn(3, 512, generator=g).to(dev)
    x[0], x[1, 5] = 0.0, math.nan
    y = L.norm_rows(x, F.PRO_RMS, eps=1e-6)
    assert bool((y[0] == 0).all()) and bool(y[1].isnan().all()) and bool(y[2].isfinite().all())


# ---- the linear ---------------------------------------------------------------------------------------------------------------------

def _operands(g, dev, M, N, K):
    x = (torch.randn(M, K, generator=g) * (0.2 + torch.randn(K, generator=g).abs() * 5)).to(dev)
    w = (torch.randn(N, K, generator=g) * (0.01 + 0.02 * torch.rand(N, 1, generator=g))).to(dev)
    return *_formula(x, 1), *_formula(w, 128)


def _check_linear(got, xs64, ws64, bias, base, K):
    exact, mass = xs64 @ ws64.t(), xs64.abs() @ ws64.abs().t()
    for extra in (bias, base):
        if extra is not None:
            exact, mass = exact + extra.double(), mass + extra.double().abs()
    bound = _half(got.dtype) * exact.abs() + (K + 4) * 2.0 ** -23 * mass + _least(got.dtype)
    err = (got.double() - exact).abs()
    assert bool((err <= bound).all()), ((err / bound).max().item(), err.max().item())


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 128, 128), (1, 2563, 2560), (2, 40, 144), (3, 1000, 9728), (7, 2563, 9744), (8, 19456, 256), (15, 130, 4096), (16, 257, 1152),
                                   (17, 129, 640), (31, 64, 32), (32, 300, 14336), (33, 127, 272), (63, 1030, 1024), (64, 640, 1280), (65, 640, 1280), (100, 130, 400),
                                   (128, 128, 128), (129, 300, 512), (200, 2050, 640), (257, 70, 8192), (333, 1030, 1040), (512, 5000, 384), (1100, 9000, 256), (2000, 5130, 512),
                                   (4100, 2560, 272)])
def test_linear(pkg, dev, M, N, K):
    g = torch.Generator().manual_seed(M * 7 + N + K)
    x, xs, w, ws = _operands(g, dev, M, N, K)
    x64, w64 = _values(x, xs, 1), _values(w, ws, 128)
    for dt in DT.values():
        bias = torch.randn(N, generator=g).to(dt).to(dev)
        out = torch.full((M + 1, N), 7.0, dtype=dt, device=dev)
        pkg.linear.f8_linear(x, xs, w, ws, bias, out=out[:M])
        _check_linear(out[:M], x64, w64, bias, None, K)
        assert bool((out[M] == 7.0).all())
        base = torch.randn(M, N, generator=g).to(dt).to(dev)
        acc = base.clone()
        pkg.linear.f8_linear(x, xs, w, ws, out=acc, beta=1.0)
        _check_linear(acc, x64, w64, None, base, K)
        assert torch.equal(pkg.linear.f8_linear(x, xs, w, ws, out_dtype=dt), pkg.linear.f8_linear(x, xs, w, ws, out_dtype=dt))
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("M,tiles,width", [(5, n, 128) for n in (1, 22, 23, 44, 46, 58, 69, 90, 97, 149)] + [(40, n, 128) for n in (43, 57, 73)] +
                         [(130, n, 256) for n in (1, 15, 16, 22, 23, 34, 35)] + [(482, 15, 256)])
def test_linear_with_every_number_of_ctas_to_a_tile(pkg, dev, M, tiles, width):
    """Sums of one to six CTAs and of one to four pairs, onto what is there and with a bias; widths whose last tile ends inside four columns too."""
    g = torch.Generator().manual_seed(M + tiles)
    K = 3200
    for N in (tiles * width - 120, tiles * width - 1):
        N = max(N, 1)
        x, xs, w, ws = _operands(g, dev, M, N, K)
        x64, w64 = _values(x, xs, 1), _values(w, ws, 128)
        for dt in DT.values():
            bias, base = torch.randn(N, generator=g).to(dt).to(dev), torch.randn(M + 1, N, generator=g).to(dt).to(dev)
            out = base.clone()
            pkg.linear.f8_linear(x, xs, w, ws, bias, out=out[:M], beta=1.0)
            _check_linear(out[:M], x64, w64, bias, base[:M], K)
            assert torch.equal(out[M], base[M])
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("M", [1, 20, 50, 150, 700])
def test_linear_on_strided_rows_and_into_a_slice(pkg, dev, M):
    g = torch.Generator().manual_seed(M)
    N, K = 200, 512
    x, xs, w, ws = _operands(g, dev, M, N, K)
    wide = torch.zeros(M, 3 * K, device=dev).to(F8)
    wide[:, K:2 * K] = x
    for dt in DT.values():
        for lead in (N, N + 1):              # rows of out on and off whole vectors
            out = torch.full((M, 3 * N + 2), 5.0, dtype=dt, device=dev)
            pkg.linear.f8_linear(wide[:, K:2 * K], xs, w, ws, out=out[:, lead:lead + N])
            _check_linear(out[:, lead:lead + N], _values(x, xs, 1), _values(w, ws, 128), None, None, K)
            assert bool((out[:, :lead] == 5.0).all()) and bool((out[:, lead + N:] == 5.0).all())


@pytest.mark.parametrize("M", [1, 30, 60, 130, 600])
def test_scales_of_every_size_and_codes_that_are_no_numbers(pkg, dev, M):
    """Blocks whose scales lie 2^40 apart; NaN in one row of x, and in one row of the weight, shows in that row and column alone."""
    g = torch.Generator().manual_seed(M)
    N, K = 700, 640
    x, xs, w, ws = _operands(g, dev, M, N, K)
    xs *= torch.exp2(torch.randint(-20, 21, xs.shape, generator=g).float()).to(dev)
    ws *= torch.exp2(torch.randint(-20, 21, ws.shape, generator=g).float()).to(dev)
    _check_linear(pkg.linear.f8_linear(x, xs, w, ws, out_dtype=torch.float32), _values(x, xs, 1), _values(w, ws, 128), None, None, K)
    x.view(torch.uint8)[M // 2, 300], w.view(torch.uint8)[130, 5] = 0x7F, 0xFF
    y = pkg.linear.f8_linear(x, xs, w, ws, out_dtype=torch.float32).isnan()
    want = torch.zeros_like(y)
    want[M // 2], want[:, 130] = True, True
    assert torch.equal(y, want)


# ---- rotary -------------------------------------------------------------------------------------------------------------------------

def _rotated(x, angle, scale, weight, eps, interleaved):
    """(result, |a| + |b| of each value's pair) in 64 bits; angle [B, L, half]."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = angle.shape[-1]
    i = torch.arange(half, device=x.device)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = (scale * angle.cos())[:, :, None], (scale * angle.sin())[:, :, None]
    out, size = y.clone(), y.abs()
    a, b = y[..., one], y[..., two]
    out[..., one], out[..., two] = a * c - b * s, a * s + b * c
    size[..., one] = size[..., two] = (a.abs() + b.abs()) * scale
    return out, size


def _check_rotary(got, x, angle, scale, weight, eps, interleaved):
    want, size = _rotated(x, angle, scale, weight, eps, interleaved)
    bound = _half(got.dtype) * want.abs() + (1 + _half(got.dtype)) * 40 * 2.0 ** -24 * size + _least(got.dtype)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), ((err / bound).max().item(), err.max().item())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,L,H,Hkv,D,rot", [(1, 1, 1, 1, 8, 8), (8, 1, 32, 8, 128, 128), (1, 7, 3, 1, 80, 80), (2, 100, 5, 5, 96, 48), (3, 33, 4, 2, 64, 40), (1, 50, 2, 1, 256, 256),
                                             (2, 9, 7, 1, 256, 6), (1, 20, 4, 0, 128, 0), (1, 11, 2, 2, 48, 34), (4, 600, 3, 1, 128, 96), (2, 1300, 2, 2, 72, 72)])
def test_rotary(pkg, dev, B, L, H, Hkv, D, rot, dtype):
    g = torch.Generator().manual_seed(B + L * 3 + H + D + rot)
    dt, A = DT[dtype], pkg.attention
    q = (torch.randn(B, L, H, D, generator=g) * 3).to(dt).to(dev)
    k = (torch.randn(B, L, Hkv, D, generator=g) * 3).to(dt).to(dev) if Hkv else None
    pos = torch.randint(-50, 1000000, (B, L), generator=g, dtype=torch.int32).to(dev)
    freq, _ = A.rope_frequencies(rot, device=dev)
    norm = (1 + 0.3 * torch.randn(2, D, generator=g)).to(dev)
    for interleaved in (False, True):
        for w in ((None, None), (norm[0], norm[1]), (norm[0], None)):
            angle = pos.double()[..., None] * freq
            qo, ko = A.rotary(q, k, pos, freq, interleaved=interleaved, q_norm=w[0], k_norm=w[1], eps=1e-6, scale=1.25)
            _check_rotary(qo, q, angle, 1.25, w[0], 1e-6, interleaved)
            if k is not None:
                _check_rotary(ko, k, angle, 1.25, w[1], 1e-6, interleaved)
            q1, k1 = q.clone(), None if k is None else k.clone()
            A.rotary(q1, k1, pos, freq, interleaved=interleaved, q_norm=w[0], k_norm=w[1], eps=1e-6, scale=1.25, q_out=q1, k_out=k1)      # in place
            assert torch.equal(q1, qo) and (k is None or torch.equal(k1, ko))
    if rot:
        places = torch.randint(0, 300, (3, B, L), generator=g, dtype=torch.int32).to(dev)
        axis = (torch.arange(rot // 2) % 3).to(torch.uint8).to(dev)
        angle = places.double()[axis.long()].permute(1, 2, 0) * freq
        qo, _ = A.rotary(q, None, places, freq, axis=axis)
        _check_rotary(qo, q, angle, 1.0, None, 0.0, False)


def test_rotary_on_slices_of_a_projection(pkg, dev):
    g = torch.Generator().manual_seed(4)
    B, L, H, Hkv, D = 2, 37, 6, 2, 64
    freq, scale = pkg.attention.rope_frequencies(48, scaling="bands", factor=8.0, device=dev)
    pos = torch.arange(4 * L, dtype=torch.int32, device=dev)[::1].view(4, L)[::2]         # a batch stride of its own
    for dt in DT.values():
        qkv = torch.randn(B, L, (H + 2 * Hkv) * D, generator=g).to(dt).to(dev)
        before = qkv.clone()
        q, k = qkv[..., :H * D].view(B, L, H, D), qkv[..., H * D:(H + Hkv) * D].view(B, L, Hkv, D)
        pkg.attention.rotary(q, k, pos, freq, scale=scale, q_out=q, k_out=k)
        angle = pos.double()[..., None] * freq
        _check_rotary(q, before[..., :H * D].view(B, L, H, D), angle, scale, None, 0.0, False)
        _check_rotary(k, before[..., H * D:(H + Hkv) * D].view(B, L, Hkv, D), angle, scale, None, 0.0, False)
        assert torch.equal(qkv[..., (H + Hkv) * D:], before[..., (H + Hkv) * D:])


# ---- packed attention -----------------------------------------------------------------------------------------------------------------

def _check_packed(got, q, k, v, offsets, causal, scale=None, visible=None):
    """Every head of every sequence; `visible(values)`: what of v counts, where some of it is no number."""
    rows, H, D = q.shape
    ratio = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    for s, e in zip(offsets[:-1], offsets[1:]):
        n = e - s
        seen = torch.ones(n, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril()
        for h in range(H):
            want, a, rest = _reference(q[s:e, h].double(), k[s:e, h // ratio].double(), v[s:e, h // ratio].double(), seen, scale)
            _check_attention(got[s:e, h], want, a, rest, _half(q.dtype))


def _packed(g, dev, dt, rows, H, Hkv, D):
    return tuple((torch.randn(rows, h, D, generator=g) * s).to(dt).to(dev) for h, s in ((H, 2.0), (Hkv, 1.5), (Hkv, 1.0)))


def _offsets(lens, dev, first=0):
    o = [first]
    for n in lens:
        o.append(o[-1] + n)
    return o, torch.tensor(o, dtype=torch.int32, device=dev)


PACKS = [([1], 1, 1, 8), ([5, 1, 0, 3], 2, 1, 64), ([64, 63, 65], 3, 3, 64), ([128], 1, 1, 128), ([127, 0, 129, 1], 4, 1, 128), ([256, 257], 2, 2, 40), ([300, 20], 6, 2, 80),
         ([77] * 9, 12, 12, 64), ([0, 0, 500], 8, 2, 128), ([1000], 5, 1, 96), ([100, 400, 31], 32, 2, 64), ([33, 200], 40, 2, 72), ([150, 90], 7, 1, 128),
         ([70, 300], 4, 2, 160), ([257, 3], 6, 1, 256), ([2, 1, 1, 2] * 60, 4, 4, 64), ([1100, 700], 8, 8, 128), ([40], 64, 1, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,H,Hkv,D", PACKS, ids=[f"{i}" for i in range(len(PACKS))])
def test_packed_attention(pkg, dev, lens, H, Hkv, D, causal, dtype):
    g = torch.Generator().manual_seed(sum(lens) + H + D)
    before, behind = 3, 7
    o, offsets = _offsets(lens, dev, before)
    rows = o[-1] + behind
    q, k, v = _packed(g, dev, DT[dtype], rows, H, Hkv, D)
    for t in (k, v):                             # rows of no sequence hold what they like
        t[:before], t[o[-1]:] = math.nan, math.nan
    out = torch.full_like(q, 9.0)
    got = pkg.attention.packed_attention(q, k, v, offsets, causal=causal, out=out)
    _check_packed(got, q, k, v, o, causal)
    assert bool((out[:before] == 9.0).all()) and bool((out[o[-1]:] == 9.0).all())
    again = pkg.attention.packed_attention(q, k, v, offsets, causal=causal)
    assert torch.equal(again[before:o[-1]], got[before:o[-1]]) and bool((again[o[-1]:] == 0).all())
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_on_slices_and_onto_its_queries(pkg, dev, causal):
    g = torch.Generator().manual_seed(8)
    H, Hkv, D = 6, 2, 64
    o, offsets = _offsets([150, 0, 70, 300], dev)
    for dt in (torch.float16, torch.bfloat16):
        qkv = torch.randn(o[-1], (H + 2 * Hkv) * D, generator=g).to(dt).to(dev)
        before = qkv.clone()
        part = lambda t, a, n: t[:, a * D:(a + n) * D].view(o[-1], n, D)  # noqa: E731
        q, k, v = part(qkv, 0, H), part(qkv, H, Hkv), part(qkv, H + Hkv, Hkv)
        pkg.attention.packed_attention(q, k, v, offsets, causal=causal, out=q, scale=0.2)
        _check_packed(q, part(before, 0, H), k, v, o, causal, 0.2)
        assert torch.equal(qkv[:, H * D:], before[:, H * D:])
        one = torch.randn(o[-1], 1, D, generator=g).to(dt).to(dev)          # one head of k and v for all, heads before rows
        qt = torch.randn(H, o[-1], D, generator=g).to(dt).to(dev).transpose(0, 1)
        _check_packed(pkg.attention.packed_attention(qt, one.expand(-1, Hkv, -1), one.expand(-1, Hkv, -1), offsets, causal=causal), qt, one.expand(-1, Hkv, -1),
                      one.expand(-1, Hkv, -1), o, causal)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 1, 128), (2, 2, 64), (3, 1, 256)])
def test_what_a_row_does_not_see_does_not_reach_it(pkg, dev, H, Hkv, D, dtype):
    """NaN and infinities in k and v: of other sequences never, of later tokens only from their own row on."""
    g = torch.Generator().manual_seed(D)
    o, offsets = _offsets([200, 130, 300, 64], dev)
    for causal in (True, False):
        q, k, v = _packed(g, dev, DT[dtype], o[-1], H, Hkv, D)
        clean = pkg.attention.packed_attention(q, k, v, offsets, causal=causal)
        bad = [o[0] + 150, o[2] + 130, o[2] + 299]
        v[bad[0], :, 5], v[bad[1], :, 17], v[bad[2], :, 0] = math.nan, math.inf, -math.inf
        got = pkg.attention.packed_attention(q, k, v, offsets, causal=causal)
        fine = torch.ones_like(got, dtype=torch.bool)
        fine[bad[0] if causal else o[0]:o[1], :, 5] = False
        fine[bad[1] if causal else o[2]:o[3], :, 17] = False
        fine[bad[2] if causal else o[2]:o[3], :, 0] = False
        assert torch.equal(got[fine], clean[fine]) and not bool(got[~fine].isfinite().any())
        k[o[1] + 100] = math.nan                 # a key: the rows that see it have no number at all
        got = pkg.attention.packed_attention(q, k, v, offsets, causal=causal)
        fine[o[1] + 100 if causal else o[1]:o[2]] = False
        assert torch.equal(got[fine], clean[fine]) and bool(got[o[1] + 100:o[2]].isnan().all())


def test_offsets_outside_the_rows(pkg, dev):
    """They end where the rows do; falling ones are empty sequences."""
    g = torch.Generator().manual_seed(1)
    for D in (64, 256):
        q, k, v = _packed(g, dev, torch.float16, 200, 2, 1, D)
        want = pkg.attention.packed_attention(q, k, v, torch.tensor([0, 100, 200], dtype=torch.int32, device=dev))
        assert torch.equal(pkg.attention.packed_attention(q, k, v, torch.tensor([-5, 100, 5000], dtype=torch.int32, device=dev)), want)
        got = pkg.attention.packed_attention(q, k, v, torch.tensor([0, 100, 50], dtype=torch.int32, device=dev))
        assert torch.equal(got[:100], want[:100]) and bool((got[100:] == 0).all())


@pytest.mark.parametrize("B", [1, 5, 40])
def test_more_items_than_a_launch_lists(pkg, dev, B):
    """Many heads of one row tile each: 512 groups fill a launch's lists with 37 tiles of 256 tokens; the next ones go to a second launch and a third."""
    g = torch.Generator().manual_seed(B)
    H, D = 512, 8
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    rows = 256 * (2 * (128 * sms // H) + 3) + 100
    o = [0, *sorted(int(c) for c in torch.randint(0, rows + 1, (B - 1,), generator=g)), rows]
    q, k, v = (torch.randn(rows, H, D, device=dev, dtype=torch.float16) for _ in range(3))
    offsets = torch.tensor(o, dtype=torch.int32, device=dev)
    got = pkg.attention.packed_attention(q, k, v, offsets)
    for s, e in zip(o[:-1], o[1:]):              # a few heads and rows of every sequence, its ends among them
        at = sorted({s, min(s + 300, e - 1), (s + e) // 2, e - 1}) if e > s else []
        for h in (0, 255, 511):
            for i in at:
                seen = torch.ones(1, i + 1 - s, dtype=torch.bool, device=dev)
                want, a, rest = _reference(q[i:i + 1, h].double(), k[s:i + 1, h].double(), v[s:i + 1, h].double(), seen, D ** -0.5)
                _check_attention(got[i:i + 1, h], want, a, rest, _half(q.dtype))
    again = q.clone()                            # onto the queries, launch after launch
    pkg.attention.packed_attention(again, k, v, offsets, out=again)
    assert torch.equal(again, got) and pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 64), (8, 2, 128), (3, 1, 96)])
def test_every_length_around_a_tiles_end(pkg, dev, H, Hkv, D, causal):
    """One sequence of each length at which a tile of 128 or 256 rows, or of 128 keys, begins or ends, beside a long one that keeps the tiles full."""
    g = torch.Generator().manual_seed(H)
    ratio = H // Hkv
    ends = sorted({n for t in (128 // ratio, 256 // ratio, 128, 256, 384) for n in (t - 1, t, t + 1)})
    q, k, v = _packed(g, dev, torch.bfloat16, 1700, H, Hkv, D)
    want = {}
    for n in ends:
        o, offsets = _offsets([n, 1700 - n], dev)
        got = pkg.attention.packed_attention(q, k, v, offsets, causal=causal)
        _check_packed(got[:n], q[:n], k[:n], v[:n], [0, n], causal)
        want[n] = got[:n].clone()
        o, offsets = _offsets([700, n], dev)     # the same rows elsewhere, and in another order of work
        moved = [torch.cat((t[-700:], t[:n])) for t in (q, k, v)]
        assert torch.equal(pkg.attention.packed_attention(*moved, offsets, causal=causal)[700:], want[n])


def test_packed_attention_agrees_with_the_other_attentions(pkg, dev):
    """One sequence without a mask is cross attention to itself; over an int8 cache the same prompt is near."""
    g = torch.Generator().manual_seed(3)
    n, H, Hkv, D = 300, 8, 2, 128
    q, k, v = _packed(g, dev, torch.float16, n, H, Hkv, D)
    _, offsets = _offsets([n], dev)
    a = pkg.attention.packed_attention(q, k, v, offsets, causal=False).double()
    b = pkg.attention.cross_attention(q[None], k[None], v[None])[0].double()
    assert float((a - b).norm() / b.norm()) < 2.0 ** -9          # both within 2^-10 of the exact rows, in the norm
    cache = pkg.attention.Kv8Cache.empty(8, Hkv, D, device=dev)
    table = torch.arange(8, dtype=torch.int32, device=dev)[None]
    pkg.attention.kv8_append(cache, k[None], v[None], table, torch.zeros(1, dtype=torch.int32, device=dev))
    c = pkg.attention.kv8_attention(q[None], cache, table, torch.tensor([n], dtype=torch.int32, device=dev))[0].double()
    a = pkg.attention.packed_attention(q, k, v, offsets).double()
    assert float((a - c).norm() / a.norm()) < 0.1


# ---- together ----------------------------------------------------------------------------------------------------------------------

def _layer(pkg, x, stream, offsets, pos, freq, scale, m):
    """One layer of a text encoder over packed prompts: what it writes, step by step."""
    L, A, F = pkg.linear, pkg.attention, pkg.ffi
    H, Hkv, D, f = m["H"], m["Hkv"], m["D"], m["f"]
    a8 = L.norm_rows(x, F.PRO_RMS, norm_w=m["norm1"], eps=1e-6, resid=stream, out_dtype=F8)
    qkv = L.f8_linear(*a8, *m["qkv"], out_dtype=x.dtype)
    rows = qkv.shape[0]
    q, k, v = (qkv[:, s * D:(s + n) * D].view(1, rows, n, D) for s, n in ((0, H), (H, Hkv), (H + Hkv, Hkv)))
    q1, k1 = A.rotary(q, k, pos, freq, q_norm=m["q_norm"], k_norm=m["k_norm"], eps=1e-6, scale=scale)
    o = A.packed_attention(q1[0], k1[0], v[0], offsets)
    o8 = L.norm_rows(o.view(rows, H * D), F.PRO_PLAIN, out_dtype=F8)
    y = L.f8_linear(*o8, *m["out"], out_dtype=x.dtype)
    b8 = L.norm_rows(y, F.PRO_RMS, norm_w=m["norm2"], eps=1e-6, resid=stream, out_dtype=F8)
    mid = L.f8_linear(*b8, *m["up"], out_dtype=x.dtype)
    c8 = L.norm_rows(mid, F.PRO_SWIGLU, K=f, up_offset=f, out_dtype=F8)
    z = L.f8_linear(*c8, *m["down"], out_dtype=x.dtype)
    return {"a8": a8, "qkv": qkv, "q1": q1, "k1": k1, "o": o, "o8": o8, "y": y, "b8": b8, "mid": mid, "c8": c8, "z": z}


def _model(pkg, g, dev, h=256, H=4, Hkv=2, D=64, f=384):
    L = pkg.linear
    pack = lambda n, k: L.f8_requant((torch.randn(n, k, generator=g) * 0.05).to(dev))  # noqa: E731
    near1 = lambda n: (1 + 0.2 * torch.randn(n, generator=g)).to(dev)  # noqa: E731
    return {"H": H, "Hkv": Hkv, "D": D, "f": f, "qkv": pack((H + 2 * Hkv) * D, h), "out": pack(h, H * D), "up": pack(2 * f, h), "down": pack(h, f), "norm1": near1(h),
            "norm2": near1(h), "q_norm": near1(D), "k_norm": near1(D)}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens", [[1], [9, 40], [130, 0, 77, 20]])
def test_a_text_encoders_layer(pkg, dev, lens, dtype):
    """The run that the operators are for, each step against its formula from what it was given."""
    g = torch.Generator().manual_seed(sum(lens))
    dt = DT[dtype]
    m = _model(pkg, g, dev)
    o, offsets = _offsets(lens, dev)
    rows, H, Hkv, D, f = o[-1], m["H"], m["Hkv"], m["D"], m["f"]
    x, stream = ((torch.randn(rows, 256, generator=g) * 2).to(dt).to(dev) for _ in range(2))
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens])[None].to(dev)
    freq, scale = pkg.attention.rope_frequencies(D, device=dev)
    s1 = (x.float() + stream.float()).to(dt)
    r = _layer(pkg, x, stream, offsets, pos, freq, scale, m)
    n = s1.double()
    _check_rows(*r["a8"], n / (n.square().mean(1, keepdim=True) + 1e-6).sqrt() * m["norm1"].double())
    for name, src in (("qkv", "a8"), ("out", "o8"), ("up", "b8"), ("down", "c8")):
        got = r[{"qkv": "qkv", "out": "y", "up": "mid", "down": "z"}[name]]
        _check_linear(got, _values(*r[src], 1), _values(*m[name], 128), None, None, r[src][0].shape[1])
    angle = pos.double()[..., None] * freq
    q, k, v = (r["qkv"][:, s * D:(s + n) * D].view(1, rows, n, D) for s, n in ((0, H), (H, Hkv), (H + Hkv, Hkv)))
    _check_rotary(r["q1"], q, angle, scale, m["q_norm"], 1e-6, False)
    _check_rotary(r["k1"], k, angle, scale, m["k_norm"], 1e-6, False)
    _check_packed(r["o"], r["q1"][0], r["k1"][0], v[0], o, True)
    s2 = (r["y"].float() + s1.float()).to(dt)
    assert torch.equal(stream, s2)
    n = s2.double()
    _check_rows(*r["b8"], n / (n.square().mean(1, keepdim=True) + 1e-6).sqrt() * m["norm2"].double())
    a, b = r["mid"][:, :f].double(), r["mid"][:, f:].double()
    _check_rows(*r["c8"], a / (1 + torch.exp(-a)) * b, 2.0 ** -20)


def test_a_linear_as_a_model_holds_it(pkg, dev):
    g = torch.Generator().manual_seed(2)
    w = (torch.randn(300, 256, generator=g) * 0.05).to(dev)
    for dt in DT.values():
        lin = pkg.linear.F8Linear.from_float(w, torch.randn(300, generator=g).to(dt).to(dev))
        x = torch.randn(10, 256, generator=g).to(dt).to(dev)
        codes, s = pkg.linear.norm_rows(x, pkg.ffi.PRO_PLAIN, out_dtype=F8)
        assert torch.equal(lin.forward(x), pkg.linear.f8_linear(codes, s, lin.weight, lin.scale, lin.bias, out_dtype=dt))
        stream, nw = torch.randn(10, 256, generator=g).to(dt).to(dev), torch.ones(256, device=dev)
        kept = stream.clone()
        y = lin.forward(x, prologue=pkg.ffi.PRO_RMS, norm_w=nw, eps=1e-6, resid=stream)
        codes, s = pkg.linear.norm_rows(x, pkg.ffi.PRO_RMS, norm_w=nw, eps=1e-6, resid=kept, out_dtype=F8)
        assert torch.equal(stream, kept) and torch.equal(y, pkg.linear.f8_linear(codes, s, lin.weight, lin.scale, lin.bias, out_dtype=dt))


@pytest.mark.parametrize("lens", [[1], [60, 200], [700, 500]])
def test_replayed_from_a_graph_two_streams_at_once_and_ordinary_launches(pkg, dev, lens):
    g = torch.Generator().manual_seed(5)
    m = _model(pkg, g, dev, h=512, f=1024)
    o, offsets = _offsets(lens, dev)
    rows = o[-1]
    x, stream = (torch.randn(rows, 512, generator=g).bfloat16().to(dev) for _ in range(2))
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens])[None].to(dev)
    freq, scale = pkg.attention.rope_frequencies(m["D"], device=dev)
    run = lambda s: _layer(pkg, x, s, offsets, pos, freq, scale, m)["z"]  # noqa: E731
    s0 = stream.clone()
    want = run(s0)
    side = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            outs.append(run(stream.clone()))
    torch.cuda.synchronize()
    assert all(torch.equal(z, want) for z in outs)
    was = pkg.linear.set_gemm_cluster_limit(4)
    try:
        assert torch.equal(run(stream.clone()), want)
    finally:
        pkg.linear.set_gemm_cluster_limit(was)
    with torch.cuda.stream(side[0]):
        s1 = stream.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[0]):
            z = run(s1)
        for _ in range(2):
            s1.copy_(stream)
            z.zero_()
            graph.replay()
            side[0].synchronize()
            assert torch.equal(z, want) and torch.equal(s1, s0)
    assert pkg.linear.kernel_status() == 0


def test_arguments_that_python_refuses(pkg, dev):
    L, A, F = pkg.linear, pkg.attention, pkg.ffi
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    c = lambda *s: torch.zeros(*s, device=dev).to(F8)  # noqa: E731
    bad = [lambda: A.packed_attention(h(4, 3, 64), h(4, 2, 64), h(4, 2, 64), i(2)), lambda: A.packed_attention(h(4, 2, 64), h(5, 2, 64), h(5, 2, 64), i(2)),
           lambda: A.packed_attention(h(4, 2, 64), h(4, 2, 64), h(4, 2, 64), i(2).long()), lambda: A.packed_attention(f(4, 2, 64), f(4, 2, 64), f(4, 2, 64), i(2)),
           lambda: A.packed_attention(h(4, 2, 64), h(4, 2, 64), h(4, 2, 64).bfloat16(), i(2)), lambda: A.packed_attention(h(4, 2, 64), h(4, 2, 64), h(4, 2, 64), i(2), out=h(4, 2, 32)),
           lambda: A.packed_attention(h(4, 2, 64), h(4, 2, 64), h(4, 2, 64), i(0)),
           lambda: A.rotary(h(1, 2, 3, 64), None, i(1, 3), f(32).double()), lambda: A.rotary(h(1, 2, 3, 64), None, i(1, 2), f(32)),
           lambda: A.rotary(h(1, 2, 3, 64), None, i(1, 2), f(33).double()), lambda: A.rotary(h(1, 2, 3, 64), None, i(2, 1, 2), f(32).double()),
           lambda: A.rotary(h(1, 2, 3, 64), h(1, 2, 3, 32), i(1, 2), f(8).double()), lambda: A.rotary(h(1, 2, 3, 64), None, i(1, 2), f(32).double(), q_norm=f(32)),
           lambda: A.rotary(h(1, 2, 3, 64), None, i(1, 2), f(32).double(), k_out=h(1, 2, 3, 64)),
           lambda: L.norm_rows(f(4, 64), norm_w=f(32)), lambda: L.norm_rows(f(4, 64), resid=f(4, 32)), lambda: L.norm_rows(f(4, 64), resid=h(4, 64)),
           lambda: L.norm_rows(f(4, 64), resid_out=f(4, 64)), lambda: L.norm_rows(f(4, 64), F.PRO_SWIGLU, K=64, up_offset=16), lambda: L.norm_rows(f(4, 64), K=80),
           lambda: L.norm_rows(f(4, 64), out=f(4, 32)), lambda: L.norm_rows(f(4, 64), scales=f(4, 1)), lambda: L.norm_rows(f(64, 4).t()),
           lambda: L.f8_linear(c(4, 64), f(4, 2), c(8, 64), f(1, 1)), lambda: L.f8_linear(c(4, 64), f(4, 1), c(8, 64), f(2, 1)), lambda: L.f8_linear(f(4, 64), f(4, 1), c(8, 64), f(1, 1)),
           lambda: L.f8_linear(c(4, 64), f(4, 1), c(8, 64), f(1, 1), beta=1.0), lambda: L.f8_linear(c(4, 64), f(4, 1), c(8, 64), f(1, 1), f(8), out_dtype=torch.float16),
           lambda: L.f8_linear(c(4, 64), f(4, 1), c(8, 80), f(1, 1)), lambda: L.f8_dequant(c(4, 64), f(4, 1)), lambda: L.f8_dequant(c(4, 64), f(4, 1), rows=2),
           lambda: L.f8_requant(f(64, 4).t())]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was taken")
    for call in (lambda: L.norm_rows(f(4, 24), out_dtype=F8), lambda: L.norm_rows(f(4, 64)[:, 1:], K=56), lambda: L.norm_rows(f(4, 64), F.PRO_SILU),
                 lambda: L.f8_linear(c(4, 24), f(4, 1), c(8, 24), f(1, 1)), lambda: A.packed_attention(h(4, 2, 36), h(4, 2, 36), h(4, 2, 36), i(2)),
                 lambda: A.rotary(h(1, 2, 3, 264), None, i(1, 2), f(32).double())):
        with pytest.raises(pkg.ffi.GpuKernelError):
            call()


def test_on_another_stream_than_the_tensors_own(pkg, dev):
    """Calls go to the current stream, whichever made the tensors."""
    L, A, F = pkg.linear, pkg.attention, pkg.ffi
    g = torch.Generator().manual_seed(6)
    x = torch.randn(200, 256, generator=g).bfloat16().to(dev)
    w, ws = L.f8_requant((torch.randn(512, 256, generator=g) * 0.1).to(dev))
    freq, _ = A.rope_frequencies(64, device=dev)
    pos = torch.arange(200, dtype=torch.int32, device=dev)[None]
    _, offsets = _offsets([150, 50], dev)

    def run():
        y = L.f8_linear(*L.norm_rows(x, F.PRO_RMS, eps=1e-6, out_dtype=F8), w, ws)
        q, k = A.rotary(y[:, :256].view(1, 200, 4, 64), y[:, 256:384].view(1, 200, 2, 64), pos, freq)
        return A.packed_attention(q[0], k[0], y[:, 384:].view(200, 2, 64), offsets)
    want = run()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_of_rows_beyond_32_bits(pkg, dev):
    """Rows whose elements lie further than 2^31 from the first: 600 000 rows of 32 heads of 128."""
    g = torch.Generator().manual_seed(12)
    rows, H, D = 600000, 32, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    q = torch.zeros(rows, H, D, dtype=torch.bfloat16, device=dev)
    tail = (torch.randn(300, H, D, generator=g) * 2).bfloat16().to(dev)
    q[-300:] = tail
    kv = torch.zeros(rows, 1, D, dtype=torch.bfloat16, device=dev)
    kv[-300:] = torch.randn(300, 1, D, generator=g).bfloat16().to(dev)
    small = [0, 250, 300]
    offsets = torch.tensor([rows - 300 + n for n in small], dtype=torch.int32, device=dev)      # the rows before belong to no sequence
    pos = torch.arange(rows, dtype=torch.int32, device=dev)[None]
    freq, _ = pkg.attention.rope_frequencies(D, device=dev)
    turned, _ = pkg.attention.rotary(q[None], None, pos, freq)
    want, _ = pkg.attention.rotary(tail[None], None, pos[:, -300:].contiguous(), freq)
    assert torch.equal(turned[0, -300:], want[0])
    out = pkg.attention.packed_attention(turned[0], kv, kv, offsets, out=turned[0])
    ref = pkg.attention.packed_attention(want[0], kv[-300:].contiguous(), kv[-300:].contiguous(), torch.tensor(small, dtype=torch.int32, device=dev))
    assert torch.equal(out[-300:], ref) and bool((out[:-300] == 0).all())
    del turned, out
    y = pkg.linear.norm_rows(q.view(rows, H * D), pkg.ffi.PRO_RMS, eps=1e-6)
    z = pkg.linear.norm_rows(tail.view(300, H * D), pkg.ffi.PRO_RMS, eps=1e-6)
    assert torch.equal(y[-300:], z) and bool((y[:-300] == 0).all())
    del y
    codes, s = pkg.linear.norm_rows(q.view(rows, H * D), pkg.ffi.PRO_PLAIN, out_dtype=F8)
    w, ws = pkg.linear.f8_requant((torch.randn(256, H * D, generator=g) * 0.05).to(dev))
    got = pkg.linear.f8_linear(codes, s, w, ws)
    _check_linear(got[-300:], _values(codes[-300:], s[-300:], 1), _values(w, ws, 128), None, None, H * D)      # (fewer rows add up in another order)
    assert bool((got[:-300] == 0).all())


def test_nothing_to_do(pkg, dev):
    L, A, F = pkg.linear, pkg.attention, pkg.ffi
    z = torch.zeros(0, 128, device=dev)
    codes, s = L.norm_rows(z, out_dtype=F8)
    assert codes.shape == (0, 128) and s.shape == (0, 1)
    w, ws = L.f8_requant(torch.ones(8, 128, device=dev))
    assert L.f8_linear(codes, s, w, ws).shape == (0, 8)
    assert L.f8_linear(*L.norm_rows(torch.ones(2, 128, device=dev), F.PRO_PLAIN, out_dtype=F8), w[:0], ws[:0]).shape == (2, 0)
    h = torch.zeros(0, 2, 64, dtype=torch.float16, device=dev)
    assert A.packed_attention(h, h, h, torch.zeros(3, dtype=torch.int32, device=dev)).shape == (0, 2, 64)
    h = torch.full((5, 2, 64), 2.0, dtype=torch.float16, device=dev)
    assert bool((A.packed_attention(h, h, h, torch.zeros(1, dtype=torch.int32, device=dev)) == 0).all())
    q, k = A.rotary(h.view(5, 1, 2, 64)[:0], None, torch.zeros(0, 1, dtype=torch.int32, device=dev), torch.zeros(32, dtype=torch.float64, device=dev))
    assert q.shape == (0, 1, 2, 64) and k is None
