"""Arguments that the attention and 4-bit entry points refuse, before a device is touched (no GPU needed)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

S = (C.c_int64 * 12)(*[64] * 12)


def _append(lib, dtype=2, B=1, L=1, Hkv=2, D=64, T=64, pages=4, max_pages=4, k=16, strides=S):
    return lib.gpu_kv8_append(dtype, k, 16, strides, 16, 16, 16, 16, 16, 4, 16, 0, B, L, Hkv, D, T, pages, max_pages, 0)


def _attention(lib, dtype=2, B=1, Lq=1, H=4, Hkv=2, D=64, T=64, pages=4, max_pages=4, q=16, strides=S):
    return lib.gpu_kv8_attention(dtype, q, 16, strides, 16, 16, 16, 16, 16, 4, 16, 0, 1, B, Lq, H, Hkv, D, T, pages, max_pages, 1.0, 0)


def _dequant(lib, dtype=0, B=1, rows=4, Hkv=2, D=64, T=64, pages=4, max_pages=4, k=32):
    return lib.gpu_kv8_dequant(dtype, 16, 16, 16, 16, 16, 4, 16, k, 32, B, rows, Hkv, D, T, pages, max_pages, 0)


def _cross(lib, dtype=2, B=1, Lq=1, Lkv=5, H=4, Hkv=2, D=64, q=16, k=16, strides=S):
    return lib.gpu_cross_attention(dtype, q, k, 16, 16, strides, 0, 0, 0, B, Lq, Lkv, H, Hkv, D, 1.0, 0)


def _w4(lib, dtype=2, sdt=1, odt=2, beta=0.0, M=1, N=8, K=64, G=32, x=16, W=16, x_stride=64):
    return lib.gpu_w4_linear(dtype, x, x_stride, W, sdt, 16, 0, 0, odt, 16, 8, beta, M, N, K, G, 0)


odd = (C.c_int64 * 12)(*[64, 64, 60] * 4)


@pytest.mark.parametrize("call,kw,code", [
    (_append, dict(dtype=3), -4), (_append, dict(T=48), -206), (_append, dict(D=72), -1), (_append, dict(D=272), -1), (_append, dict(Hkv=0), -1),
    (_append, dict(B=-1), -1), (_append, dict(k=8), -5), (_append, dict(k=0), -5), (_append, dict(strides=odd), -5), (_append, dict(max_pages=1 << 30), -1),
    (_append, dict(L=0), 0), (_append, dict(B=0), 0),
    (_attention, dict(dtype=0), -4), (_attention, dict(T=8), -206), (_attention, dict(D=40), -1), (_attention, dict(H=5), -1), (_attention, dict(H=0), -1),
    (_attention, dict(q=8), -5), (_attention, dict(strides=odd), -5), (_attention, dict(max_pages=1 << 28, T=128), -1), (_attention, dict(Lq=0), 0),
    (_attention, dict(Lq=-1), -1), (_attention, dict(pages=-1), -1),
    (_dequant, dict(dtype=7), -4), (_dequant, dict(T=0), -206), (_dequant, dict(k=4), -5), (_dequant, dict(rows=0), 0), (_dequant, dict(rows=1 << 60), -1),
    (_cross, dict(dtype=0), -4), (_cross, dict(D=36), -1), (_cross, dict(D=264), -1), (_cross, dict(H=6, Hkv=4), -1), (_cross, dict(k=0), -5),
    (_cross, dict(q=4), -5), (_cross, dict(strides=odd), -5), (_cross, dict(strides=None), -5), (_cross, dict(Lq=0), 0), (_cross, dict(Lkv=-1), -1),
    (_w4, dict(G=48), -1), (_w4, dict(K=0), -1), (_w4, dict(K=96, G=64), -1), (_w4, dict(dtype=3), -4), (_w4, dict(sdt=0), -4), (_w4, dict(odt=1), -4),
    (_w4, dict(beta=2.0), -207), (_w4, dict(x=8), -5), (_w4, dict(W=8), -5), (_w4, dict(M=0), 0), (_w4, dict(N=0), 0), (_w4, dict(M=2, x_stride=32), -5),
    (_w4, dict(M=-1), -1)])
def test_codes(pkg, call, kw, code):
    assert call(pkg.lib, **kw) == code


def test_packer_codes(pkg):
    lib = pkg.lib
    assert lib.gpu_w4_requant(2, 16, 64, 16, 1, 16, 0, 4, 64, 16, 0) == -1
    assert lib.gpu_w4_requant(2, 16, 64, 16, 0, 16, 0, 4, 64, 32, 0) == -4
    assert lib.gpu_w4_requant(2, 8, 64, 16, 1, 16, 0, 4, 64, 32, 0) == -5
    assert lib.gpu_w4_requant(2, 16, 60, 16, 1, 16, 0, 4, 64, 32, 0) == -5
    assert lib.gpu_w4_requant(2, 16, 64, 16, 1, 16, 0, 0, 64, 32, 0) == 0
    assert lib.gpu_w4_dequant(9, 16, 1, 16, 0, 16, 4, 64, 32, 0) == -4
    assert lib.gpu_w4_dequant(0, 16, 1, 16, 0, 8, 4, 64, 32, 0) == -5


def test_host_tensors_are_refused(pkg):
    A, L = pkg.attention, pkg.linear
    q = torch.zeros(1, 2, 4, 64).half()
    cache = A.Kv8Cache.empty(2, 2, 64, device="cpu")
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: A.cross_attention(q, q, q), lambda: A.kv8_attention(q, cache, t, n), lambda: A.kv8_append(cache, q, q, t, n),
                 lambda: A.kv8_dequant(cache, t, n, 4), lambda: L.w4_requant(torch.zeros(4, 64)), lambda: L.w4_linear(torch.zeros(1, 64), t, q),
                 lambda: L.w4_dequant(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2).half())):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()


@pytest.mark.parametrize("call,kw", [
    (_cross, dict(Lkv=2 ** 31 - 64)), (_cross, dict(Lkv=2 ** 31 - 1)), (_cross, dict(Lq=2 ** 31 - 1, H=4, Hkv=1, D=136)), (_cross, dict(Lq=1, B=2 ** 31 - 1, H=2 ** 30, Hkv=2 ** 30)),
    (_attention, dict(Lq=2 ** 31 - 1, H=2 ** 20, Hkv=1)), (_attention, dict(Lq=1, B=2 ** 31 - 1, H=2 ** 30, Hkv=2 ** 30)),
    (_append, dict(B=2 ** 31 - 1, L=2 ** 31 - 1, Hkv=2 ** 31 - 1)),
    (_w4, dict(M=2 ** 31 - 1, x_stride=64)), (_w4, dict(M=2 ** 31 - 100, dtype=0, odt=0)), (_w4, dict(N=2 ** 31 - 1))])
def test_sizes_that_32_bits_do_not_count(pkg, call, kw):
    assert call(pkg.lib, **kw) == -1


@pytest.mark.parametrize("call,at,kw", [(_cross, 9, dict(B=2)), (_cross, 10, dict(Lq=2)), (_cross, 11, dict(H=4)), (_attention, 3, dict(B=2)), (_attention, 4, dict(Lq=2)),
                                        (_attention, 5, dict(H=4))])
def test_rows_of_the_result_in_one_place(pkg, call, at, kw):
    strides = (C.c_int64 * 12)(*S)
    strides[at] = 0
    assert call(pkg.lib, strides=strides, **kw) == -5
