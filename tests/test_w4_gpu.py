"""Linears with 4-bit weights and group scales (gpu_w4_requant, gpu_w4_dequant, gpu_w4_linear) against their formulas in 64 bits.

Packing: the scale is one f32 product and one rounding to its type, a code one f32 division and one rounding, so both are the same
numbers in every IEEE implementation and compared for equality; what the codes stand for lies within half a step of the weight.
Linear: codes and activations enter exactly, so an output is off by the rounding to its type (half a step of the value) and by the f32
sums, at most 2^-23 of the absolute terms for each of the K additions (the products' own sums may cut off instead of rounding)."""
from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _half(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def _unpack(packed, scales, zeros):
    N, groups = scales.shape
    c = torch.stack((packed & 15, packed >> 4), 2).flatten(1).double().view(N, groups, -1)
    z = 8.0 if zeros is None else zeros.double()[:, :, None]
    return ((c - z) * scales.double()[:, :, None]).view(N, -1)


def _weight(g, dev, N, K, G, sdt=torch.float16, zeros=True):
    packed = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.int32).to(torch.uint8).to(dev)
    scales = (torch.rand(N, K // G, generator=g) * 0.01 + 1e-3).to(sdt).to(dev)
    z = torch.randint(0, 16, (N, K // G), generator=g, dtype=torch.int32).to(torch.uint8).to(dev) if zeros else None
    return packed, scales, z


def _check(got, x, w, bias, base):
    exact, mass = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    for extra in (bias, base):
        if extra is not None:
            exact, mass = exact + extra.double(), mass + extra.double().abs()
    bound = _half(got.dtype) * exact.abs() + (x.shape[1] + 4) * 2.0 ** -23 * mass + (2.0 ** -24 if got.dtype == torch.float16 else 1e-37)
    err = (got.double() - exact).abs()
    assert bool((err <= bound).all()), ((err / bound).max().item(), err.max().item())


# one token to several tiles of them, ragged everywhere: rows of W (16 and 128 to a tile), K off a block of 128, every group
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K,G", [(1, 1, 32, 32), (1, 16, 128, 128), (1, 2563, 2560, 128), (2, 40, 96, 32), (3, 1000, 9728, 32), (4, 17, 64, 64),
                                     (5, 513, 4096 + 64, 64), (7, 130, 1024, 256), (8, 19456, 256, 64), (9, 33, 160, 32), (16, 257, 768, 128),
                                     (17, 129, 192, 64), (63, 127, 288, 32), (65, 640, 1280, 128), (129, 300, 512, 256), (333, 1030, 1024, 64),
                                     # several tiles to a CTA; a tile to a cluster; columns that make tiles wide and narrow
                                     (333, 13829, 320, 64), (300, 9000, 288, 32), (70, 200, 8192, 256), (40, 100, 4160, 64), (193, 2050, 640, 128), (12, 3000, 96, 32)])
def test_linear(pkg, dev, M, N, K, G, dtype):
    g = torch.Generator().manual_seed(M * 7 + N + K)
    dt = DT[dtype]
    x = (torch.randn(M, K, generator=g) * (0.2 + torch.randn(K, generator=g).abs() * 5)).to(dt).to(dev)
    for zeros, sdt in ((True, torch.float16), (False, torch.bfloat16)):
        packed, scales, z = _weight(g, dev, N, K, G, sdt, zeros)
        w = _unpack(packed, scales, z)
        bias = torch.randn(N, generator=g).to(dt).to(dev) if zeros else None
        out = torch.full((M + 1, N), 7.0, dtype=dt, device=dev)
        pkg.linear.w4_linear(x, packed, scales, z, bias, out=out[:M])
        _check(out[:M], x, w, bias, None)
        assert bool((out[M] == 7.0).all())
        base = torch.randn(M, N, generator=g).to(dt).to(dev)
        acc = base.clone()
        pkg.linear.w4_linear(x, packed, scales, z, bias, out=acc, beta=1.0)
        _check(acc, x, w, bias, base)
    if dtype != "f32":
        y = pkg.linear.w4_linear(x, packed, scales, z, None, out_dtype=torch.float32)
        assert y.dtype == torch.float32
        _check(y, x, w, None, None)


@pytest.mark.parametrize("M", [1, 6, 40])
def test_linear_on_strided_rows_and_into_a_slice(pkg, dev, M):
    g = torch.Generator().manual_seed(M)
    K, N = 512, 200
    for dt in DT.values():
        wide = torch.randn(M, 3 * K, generator=g).to(dt).to(dev)
        packed, scales, z = _weight(g, dev, N, K, 64)
        out = torch.full((M, 3 * N + 1), 5.0, dtype=dt, device=dev)
        x = wide[:, K:2 * K]
        pkg.linear.w4_linear(x, packed, scales, z, out=out[:, N:2 * N])
        _check(out[:, N:2 * N], x, _unpack(packed, scales, z), None, None)
        assert bool((out[:, :N] == 5.0).all()) and bool((out[:, 2 * N:] == 5.0).all())


@pytest.mark.parametrize("M", [1, 30])
def test_f32_rows_keep_24_bits_whatever_their_size(pkg, dev, M):
    """An f32 value is the sum of its three bf16 terms exactly: rows of very large and very small values are as good as others."""
    g = torch.Generator().manual_seed(3)
    K, N = 256, 64
    packed, scales, z = _weight(g, dev, N, K, 32)
    w = _unpack(packed, scales, z)
    for size in (1e-30, 1e-3, 1e30):
        x = (torch.randn(M, K, generator=g) * size).to(dev)
        y = pkg.linear.w4_linear(x, packed, scales, z)
        err, mass = (y.double() - x.double() @ w.t()).abs(), x.double().abs() @ w.abs().t()
        assert bool((err <= (K + 4) * 2.0 ** -23 * mass).all())
    one = torch.zeros(M, K, device=dev)
    one[:, 5] = 1.0 + 2.0 ** -23                     # a single term: nothing but its own bits, and the scale's product
    y = pkg.linear.w4_linear(one, packed, scales, z)
    assert bool(((y.double() - one.double() @ w.t()).abs() <= 2.0 ** -23 * w[:, 5].abs()).all())


@pytest.mark.parametrize("M", [1, 9, 40, 200])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("G", [32, 256])
def test_rows_up_to_the_largest_numbers(pkg, dev, M, dtype, G):
    """Activations near the type's largest number: the codes' sums stay in range where the result does. Many columns of one sign and the
    largest codes, so that a group's sum before its scale is as large as it gets."""
    g = torch.Generator().manual_seed(M)
    K, N = 512, 70
    packed, scales, z = _weight(g, dev, N, K, G)
    packed[0], z[0] = 0xFF, 0                        # every weight 15 steps
    packed[1], z[1] = 0x00, 15                       # and every one -15
    scales.mul_(0.1)                                 # sums of at most (30 + 482 x 0.03) x 15 x 0.0011 x 3.3e38 = 2.5e38
    x = torch.rand(M, K, generator=g).mul(0.02).add(0.98).mul(torch.where(torch.rand(M, 1, generator=g) < 0.5, -1.0, 1.0)).mul(3.3e38)
    x[:, 30:] *= 0.03
    x = x.to(DT[dtype]).to(dev)
    assert bool(torch.isfinite(x).all())
    w = _unpack(packed, scales, z)
    y = pkg.linear.w4_linear(x, packed, scales, z, out_dtype=torch.float32)
    assert float((x.double() @ w.t()).abs().max()) < 3.3e38
    _check(y, x, w, None, None)


@pytest.mark.parametrize("M", [1, 30])
def test_small_values_keep_their_bits(pkg, dev, M):
    """One f32 value of 2^-100 with bits in all three of its bf16 terms: nothing but the scale's product and the terms' sum is rounded."""
    g = torch.Generator().manual_seed(M)
    K, N = 256, 64
    packed, scales, z = _weight(g, dev, N, K, 32)
    w = _unpack(packed, scales, z)
    one = torch.zeros(M, K, device=dev)
    one[:, 5] = (1.0 + 2.0 ** -15 + 2.0 ** -22) * 2.0 ** -100
    y = pkg.linear.w4_linear(one, packed, scales, z)
    assert bool(((y.double() - one.double() @ w.t()).abs() <= 2.0 ** -23 * 2.0 ** -100 * w[:, 5].abs()).all())


@pytest.mark.parametrize("M", [2, 33])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_infinities_and_nan_stay_in_their_row(pkg, dev, M, dtype):
    g = torch.Generator().manual_seed(5)
    K, N = 160, 48
    packed, scales, z = _weight(g, dev, N, K, 32, zeros=False)
    packed[:] = packed | 0x99                        # codes 9..15: every weight positive
    x = torch.rand(M, K, generator=g).to(DT[dtype]).to(dev)
    x[1, 7] = float("inf")
    y = pkg.linear.w4_linear(x, packed, scales, z)
    assert bool(torch.isposinf(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2:]).all())
    x[1, 9] = float("nan")
    y = pkg.linear.w4_linear(x, packed, scales, z)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2:]).all())


@pytest.mark.parametrize("M", [1, 5, 70])
def test_columns_behind_the_last_group_are_not_read(pkg, dev, M):
    """K = 96 fills three quarters of a block: what lies behind a row of x (here NaN) takes no part."""
    g = torch.Generator().manual_seed(M)
    for dt in DT.values():
        wide = torch.full((M, 128), float("nan"), dtype=dt, device=dev)
        wide[:, :96] = torch.randn(M, 96, generator=g).to(dt).to(dev)
        packed, scales, z = _weight(g, dev, 24, 96, 32)
        y = pkg.linear.w4_linear(wide[:, :96], packed, scales, z)
        _check(y, wide[:, :96], _unpack(packed, scales, z), None, None)


def _packed_as_defined(w, G, zeros, sdt):
    g = w.float().view(w.shape[0], -1, G)
    if zeros:
        lo, hi = g.amin(2).clamp_max(0), g.amax(2).clamp_min(0)
        s = ((hi - lo) * (1 / 15)).to(sdt)
        z = torch.where(s > 0, torch.round(-lo / s.float()), 0.0).clamp(0, 15)
    else:
        s = (g.abs().amax(2) * (1 / 7)).to(sdt)
        z = torch.full(s.shape, 8.0, device=w.device)
    c = (torch.where(s[..., None] > 0, torch.round(g / s.float()[..., None]), 0.0) + z[..., None]).clamp(0, 15)
    return c.flatten(1), s, z


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("sdt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,K,G", [(1, 32, 32), (3, 96, 32), (67, 640, 64), (129, 1280, 128), (40, 768, 256), (1000, 512, 128)])
def test_packer(pkg, dev, N, K, G, dtype, sdt):
    g = torch.Generator().manual_seed(N + K)
    w = (torch.randn(N, K + 8, generator=g) * 0.02).to(DT[dtype]).to(dev)[:, :K]      # rows further apart than they are long
    w[0, :G] = 0.0                                   # a group of zeros
    if N > 2:
        w[1, :G] = w[1, :G].abs()                    # one sign only
        w[2, 0] = 3.0                                # a group with an outlier
    for zeros in (False, True):
        packed, s, z = pkg.linear.w4_requant(w, G, zero_points=zeros, scale_dtype=sdt)
        codes, s_want, z_want = _packed_as_defined(w, G, zeros, sdt)
        assert torch.equal(s, s_want) and (z is None if not zeros else torch.equal(z.float(), z_want))
        assert torch.equal(torch.stack((packed & 15, packed >> 4), 2).flatten(1).float(), codes)
        for dt in DT.values():
            back = pkg.linear.w4_dequant(packed, s, z, dtype=dt)
            want = (codes.view(N, -1, G) - z_want[..., None]) * s.float()[..., None]
            assert torch.equal(back, want.view(N, K).to(dt))
        # within half a step, and what the ends lose to the scale's rounding (seven or fifteen steps of its half step)
        step = s.double().repeat_interleave(G, 1)
        off = (pkg.linear.w4_dequant(packed, s, z).double() - w.double()).abs()
        assert bool((off <= step * (0.5 + 15 * torch.finfo(sdt).eps + (0.5 if zeros else 0)) + 1e-6 * step + (6e-8 if sdt == torch.float16 else 0)).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("zeros", [False, True])
def test_packer_on_nan_and_infinities(pkg, dev, dtype, zeros):
    """NaN stands for 0 after packing, and the other weights of its group are as without it; an infinity takes the end of the range."""
    g = torch.Generator().manual_seed(5)
    N, K, G = 67, 256, 32
    w = (torch.randn(N, K, generator=g) * 0.02).to(DT[dtype]).to(dev)
    bad = (torch.rand(N, K, generator=g) < 0.1).to(dev)
    bad[3, :G] = True                                # a group of nothing else
    packed, s, z = pkg.linear.w4_requant(torch.where(bad, torch.tensor(float("nan"), dtype=w.dtype, device=dev), w), G, zero_points=zeros)
    want = pkg.linear.w4_requant(torch.where(bad, torch.zeros_like(w), w), G, zero_points=zeros)
    assert torch.equal(packed, want[0]) and torch.equal(s, want[1]) and (z is None or torch.equal(z, want[2]))
    assert bool((pkg.linear.w4_dequant(packed, s, z)[bad] == 0).all())
    w[1, 5], w[2, 7] = float("inf"), -float("inf")
    packed, s, z = pkg.linear.w4_requant(w, G, zero_points=zeros)
    codes = torch.stack((packed & 15, packed >> 4), 2).flatten(1)
    assert int(codes[1, 5]) == 15 and int(codes[2, 7]) == 0 and float(s[1, 0]) == 65504.0 and bool(torch.isfinite(s).all())


def test_a_lora_bake_goes_there_and_back(pkg, dev):
    """Packed, read back, packed again: the same codes (the largest of a group lands on its own scale again)."""
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(256, 1024, generator=g) * 0.02).bfloat16().to(dev)
    packed, s, _ = pkg.linear.w4_requant(w, 64, scale_dtype=torch.bfloat16)
    back = pkg.linear.w4_dequant(packed, s)
    assert torch.equal(pkg.linear.w4_dequant(*pkg.linear.w4_requant(back, 64, scale_dtype=torch.bfloat16)), back)


def test_text_encoder_mlp_in_four_bits(pkg, dev):
    """The run that the operators are for: RMS norm and rotation, gate-up, SwiGLU and rotation, down onto the residual stream, weights
    packed from their rotated form. Against the same steps in 64 bits from the same codes."""
    L, F = pkg.linear, pkg.ffi
    g = torch.Generator().manual_seed(11)
    h, f = 512, 1024
    gu = L.rotate_rows_f32((torch.randn(2 * f, h, generator=g) * 0.03).to(dev))
    down = L.rotate_rows_f32((torch.randn(h, f, generator=g) * 0.03).to(dev))
    gu_w, down_w = L.w4_requant(gu, 64, zero_points=True), L.w4_requant(down, 32)
    norm = (1 + 0.1 * torch.randn(h, generator=g)).to(dev)
    for M in (1, 6, 50):
        stream = torch.randn(M, h, generator=g).to(dev)
        want = stream.double()
        a = L.rotate_rows_f32(stream, F.PRO_RMS, norm_w=norm, eps=1e-6)
        mid = L.w4_linear(a, *gu_w)
        b = L.rotate_rows_f32(mid, F.PRO_SWIGLU, K=f, up_offset=f)
        L.w4_linear(b, *down_w, out=stream, beta=1.0)
        _check(mid, a, _unpack(*gu_w), None, None)
        _check(stream, b, _unpack(*down_w), None, want)


def test_replayed_from_a_graph_and_on_another_stream(pkg, dev):
    g = torch.Generator().manual_seed(2)
    packed, scales, z = _weight(g, dev, 700, 1024, 64)
    side = torch.cuda.Stream(dev)
    for M in (1, 5, 48):
        x = torch.randn(M, 1024, generator=g).bfloat16().to(dev)
        out = torch.empty(M, 700, dtype=torch.bfloat16, device=dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            pkg.linear.w4_linear(x, packed, scales, z, out=out)
            side.synchronize()
            eager = out.clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                pkg.linear.w4_linear(x, packed, scales, z, out=out)
                pkg.linear.w4_linear(x, packed, scales, z, out=out)
            out.zero_()
            graph.replay()
            side.synchronize()
        assert torch.equal(out, eager)
        assert all(torch.equal(pkg.linear.w4_linear(x, packed, scales, z), eager) for _ in range(3))      # the same bits every time


@pytest.mark.parametrize("M", [1, 11, 40, 200])
def test_two_streams_at_once_and_ordinary_launches(pkg, dev, M):
    """Nothing is shared between calls: two at a time give what one gives. Beside a collective's kernels launches are ordinary ones."""
    g = torch.Generator().manual_seed(M)
    L = pkg.linear
    packed, scales, z = _weight(g, dev, 1500, 2048, 64)
    for dt in DT.values():
        x = torch.randn(M, 2048, generator=g).to(dt).to(dev)
        want = L.w4_linear(x, packed, scales, z)
        outs, streams = [torch.empty_like(want) for _ in range(8)], [torch.cuda.Stream(dev) for _ in range(2)]
        torch.cuda.synchronize()
        for i, out in enumerate(outs):
            with torch.cuda.stream(streams[i % 2]):
                L.w4_linear(x, packed, scales, z, out=out)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)
        was = L.set_gemm_cluster_limit(4)
        try:
            assert torch.equal(L.w4_linear(x, packed, scales, z), want)
        finally:
            L.set_gemm_cluster_limit(was)
    assert L.kernel_status() == 0


@pytest.mark.parametrize("M", [(1, 8), (34, 160)])
def test_two_host_threads_with_different_sizes(pkg, dev, M):
    """The same kernel with little and with much shared memory, launched by two threads at once: neither takes the other's limit."""
    g = torch.Generator().manual_seed(M[0])
    L, errors = pkg.linear, []
    work = []
    for m, K in zip(M, (256, 9728)):
        packed, scales, _ = _weight(g, dev, 64, K, 128, zeros=False)
        x = torch.randn(m, K, generator=g).bfloat16().to(dev)
        want = L.w4_linear(x, packed, scales)
        _check(want, x, _unpack(packed, scales, None), None, None)
        work.append((x, packed, scales, want))
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def loop(x, packed, scales, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                out = torch.empty_like(want)
                start.wait()
                for _ in range(3000):
                    L.w4_linear(x, packed, scales, out=out)
                torch.cuda.current_stream(dev).synchronize()
                assert torch.equal(out, want)
        except BaseException as e:
            errors.append(e)
    threads = [threading.Thread(target=loop, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("M", [1, 40])
def test_offsets_beyond_32_bits(pkg, dev, M):
    """A packed weight of more than 2^31 bytes: rows at its beginning and its end."""
    N, K, G = 66000, 65536, 256
    gen = torch.Generator(device=dev).manual_seed(M)
    packed = torch.empty((N, K // 2), dtype=torch.uint8, device=dev).random_(0, 256, generator=gen)
    scales = (torch.rand(N, K // G, generator=gen, device=dev) * 0.01 + 1e-3).half()
    x = torch.randn(M, K, generator=gen, device=dev).bfloat16()
    y = pkg.linear.w4_linear(x, packed, scales, out_dtype=torch.float32)
    rows = torch.cat([torch.arange(3), torch.arange(N - 200, N, 7)]).to(dev)
    _check(y[:, rows], x, _unpack(packed[rows], scales[rows], None), None, None)


def test_refusals(pkg, dev):
    L = pkg.linear
    x = torch.zeros(2, 64, device=dev)
    packed, scales, z = L.w4_requant(torch.zeros(8, 64, device=dev), 32, zero_points=True)
    for bad in (lambda: L.w4_linear(x, packed, scales.float()), lambda: L.w4_linear(x, packed.to(torch.int8), scales), lambda: L.w4_linear(x[:, :32], packed, scales),
                lambda: L.w4_linear(x, packed, scales, z.float()), lambda: L.w4_linear(x, packed, scales, z[:, :1]), lambda: L.w4_linear(x, packed, scales, beta=1.0),
                lambda: L.w4_linear(x, packed, scales, bias=torch.zeros(7, device=dev)), lambda: L.w4_linear(x, packed, scales, out=torch.zeros(2, 7, device=dev)),
                lambda: L.w4_linear(x.t(), packed, scales), lambda: L.w4_linear(x, packed.cpu(), scales), lambda: L.w4_requant(x, 24),
                lambda: L.w4_requant(x, 128), lambda: L.w4_requant(x.t(), 32), lambda: L.w4_dequant(packed, scales[:4])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(pkg.GpuKernelError):          # beta neither 0 nor 1; out in a third type
        L.w4_linear(x, packed, scales, out=torch.zeros(2, 8, device=dev), beta=0.5)
    with pytest.raises(pkg.GpuKernelError):
        L.w4_linear(x.half(), packed, scales, out=torch.zeros(2, 8, dtype=torch.bfloat16, device=dev))
    with pytest.raises(pkg.GpuKernelError, match="-5"):
        L.w4_linear(torch.zeros(2, 68, device=dev)[:, 1:65], packed, scales)
    assert L.w4_linear(x[:0], packed, scales).shape == (0, 8)
