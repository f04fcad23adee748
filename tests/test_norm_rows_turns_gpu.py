"""gpu_norm_rows where there are more rows than the CTAs of one turn take, up to numbers of rows near 2^31: each row is what it is in a call of fewer rows."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
PART, SHIFTS = 1 << 20, 1031


def _free(dev, gib):
    if torch.cuda.mem_get_info(dev)[0] < gib << 30:
        pytest.skip(f"needs {gib} GB")


# f32 rows, and 16-bit ones of more than 8192 columns, have no next row on its way: one turn up to 2^19 rows. One warp, several and 32 warps to a row; more than 2^30 rows,
# where two turns' row numbers would leave 32 bits
@pytest.mark.parametrize("M,K,dt,out_dt,gib", [((1 << 20) + 4321, 8, torch.float32, torch.float32, 1), ((1 << 19) + 5, 1040, torch.float32, F8, 5),
                                               ((1 << 19) + 1029, 8208, torch.bfloat16, F8, 16), ((1 << 30) + 12345, 8, torch.float32, torch.bfloat16, 56)])
def test_rows_of_every_turn(pkg, dev, M, K, dt, out_dt, gib):
    _free(dev, gib)
    L, F = pkg.linear, pkg.ffi
    g = torch.Generator(device=dev).manual_seed(K)
    n = min(PART, (1 << 31) // (K * dt.itemsize) // 8)
    base = torch.randn(n + SHIFTS, K, device=dev, generator=g, dtype=torch.float32).to(dt)
    w = 1 + 0.3 * torch.randn(K, device=dev, generator=g)
    want = L.norm_rows(base, F.PRO_RMS, norm_w=w, eps=1e-6, out_dtype=out_dt)      # few rows: one turn
    x = torch.empty(M, K, dtype=dt, device=dev)
    for i, at in enumerate(range(0, M, n)):
        x[at:at + n] = base[i % SHIFTS:i % SHIFTS + min(n, M - at)]
    got = L.norm_rows(x, F.PRO_RMS, norm_w=w, eps=1e-6, out_dtype=out_dt)
    del x
    bits = lambda t: t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.dtype.itemsize])  # noqa: E731
    for a, b in zip(got, want) if out_dt == F8 else ((got, want),):
        for i, at in enumerate(range(0, M, n)):
            rows = min(n, M - at)
            assert torch.equal(bits(a[at:at + rows]), bits(b[i % SHIFTS:i % SHIFTS + rows])), (at, rows)
    assert L.kernel_status() == 0


def test_the_stream_in_every_turn(pkg, dev):
    """In place, onto the stream: a turn's rows are read before they are written, by their CTA alone."""
    _free(dev, 12)
    L, F = pkg.linear, pkg.ffi
    g = torch.Generator(device=dev).manual_seed(1)
    M, K, n = (1 << 19) + 777, 520, 1 << 17
    x, stream = (torch.randn(M, K, device=dev, generator=g) for _ in range(2))
    want = [(x[at:at + n] + stream[at:at + n], None) for at in range(0, M, n)]
    want = [(s, L.norm_rows(s, F.PRO_RMS, eps=1e-6)) for s, _ in want]
    y = L.norm_rows(x, F.PRO_RMS, eps=1e-6, resid=stream)
    for i, at in enumerate(range(0, M, n)):
        assert torch.equal(stream[at:at + n], want[i][0]) and torch.equal(y[at:at + n], want[i][1])
