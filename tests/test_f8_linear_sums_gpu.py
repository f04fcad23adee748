"""gpu_f8_linear's sums in f32, held to what its own order of additions may lose: a block's 128 products are exact and their sum is off by at most 2^-23 of their absolute sum for each of
132 additions (128 terms, the four instructions of a block); over the blocks and the CTAs that share a tile's K each addition, and the scale's product, is off by 2^-24 of the absolute sum
so far. With the absolute sum of all products times scales, `mass`, that is (132 + (blocks + 10) / 2) 2^-23 mass, and 2^-24 of the result for its way out."""
from __future__ import annotations

import pytest
import torch

from test_encoder_layer_gpu import _operands, _values


def _bound(exact, mass, K):
    blocks = -(-K // 128)
    return (132 + (blocks + 10) / 2) * 2.0 ** -23 * mass + 2.0 ** -24 * exact.abs() + 1e-37


@pytest.mark.gpu
# one CTA to a tile's K, two to six of them; pairs alone, and two to four
@pytest.mark.parametrize("M,N,K", [(1, 2563, 9728), (7, 40000, 2560), (16, 2560, 14336), (33, 8000, 3200), (40, 130, 3200), (64, 640, 32768), (65, 257, 9728), (130, 4000, 3200),
                                   (130, 8000, 3200), (300, 1030, 16400), (700, 5130, 2560), (2100, 2560, 1040)])
def test_sums(pkg, dev, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    x, xs, w, ws = _operands(g, dev, M, N, K)
    xs *= torch.exp2(torch.randint(-3, 4, xs.shape, generator=g).float()).to(dev)
    x64, w64 = _values(x, xs, 1), _values(w, ws, 128)
    exact, mass = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    bound = _bound(exact, mass, K)
    got = pkg.linear.f8_linear(x, xs, w, ws, out_dtype=torch.float32).double()
    assert bool(((got - exact).abs() <= bound).all()), ((got - exact).abs() / bound).max().item()
    base = torch.randn(M, N, generator=g).to(dev)
    got = pkg.linear.f8_linear(x, xs, w, ws, out=base.clone(), beta=1.0).double()
    exact, bound = exact + base.double(), bound + 2.0 ** -24 * (mass + 2 * base.double().abs())
    assert bool(((got - exact).abs() <= bound).all()), ((got - exact).abs() / bound).max().item()
    assert pkg.linear.kernel_status() == 0


@pytest.mark.parametrize("M,N,K", [(1, 2563, 9728), (40, 130, 3200), (130, 257, 9728)])
def test_the_bound_finds_wrong_sums(M, N, K):
    """Mistakes put into the 64-bit sums (no GPU needed): a block's scale a tenth off; the parts of three CTAs rounded to bf16 before they are added."""
    g = torch.Generator().manual_seed(M + N + K)
    x, xs, w, ws = _operands(g, "cpu", M, N, K)
    x64, w64 = _values(x, xs, 1), _values(w, ws, 128)
    exact, mass = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    at = slice(K // 256 * 128, K // 256 * 128 + 128)
    wrong = exact + 0.1 * (x64[:, at] @ w64[:, at].t())
    assert ((wrong - exact).abs() > _bound(exact, mass, K)).double().mean() > 0.5
    parts = [(a @ b.t()).bfloat16().double() for a, b in zip(x64.chunk(3, 1), w64.chunk(3, 1))]
    assert bool(((sum(parts) - exact).abs() > _bound(exact, mass, K)).any())
