"""Arguments that the entry points of a text encoder's layer refuse, before a device is touched, and the frequencies of rotary positions (no GPU needed)."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

S = (C.c_int64 * 12)(*[64] * 12)
odd = (C.c_int64 * 12)(*[64, 60] * 6)


def _norm(lib, dtype=2, pro=1, x=16, xs=128, up=0, resid=16, resid_stride=128, resid_out=16, ros=128, w=16, odt=3, out=16, os=128, scales=16, M=2, K=128):
    return lib.gpu_norm_rows(dtype, pro, x, xs, up, resid, resid_stride, resid_out, ros, w, 1e-6, odt, out, os, scales, M, K, 0)


def _linear(lib, x=16, x_stride=128, xs=16, W=16, ws=16, odt=2, out=16, out_stride=8, beta=0.0, M=2, N=8, K=128):
    return lib.gpu_f8_linear(x, x_stride, xs, W, ws, 0, odt, out, out_stride, beta, M, N, K, 0)


def _requant(lib, dtype=0, w=16, stride=128, codes=16, N=4, K=128):
    return lib.gpu_f8_requant(dtype, w, stride, codes, 16, N, K, 0)


def _dequant(lib, dtype=0, codes=16, rows=128, out=16, N=4, K=128):
    return lib.gpu_f8_dequant(dtype, codes, 16, rows, out, N, K, 0)


def _packed(lib, dtype=2, q=16, k=16, strides=S, offsets=16, B=1, rows=4, H=4, Hkv=2, D=64):
    return lib.gpu_packed_attention(dtype, q, k, 16, 16, strides, offsets, 1, B, rows, H, Hkv, D, 1.0, 0)


def _rotary(lib, dtype=2, q=16, k=16, q_out=16, strides=S, pos=16, axes=1, axis=0, freq=16, rot=64, q_norm=0, B=1, L=2, H=4, Hkv=2, D=64):
    return lib.gpu_rotary(dtype, q, k, q_out, 16, strides, pos, 2, 2, axes, axis, freq, rot, 0, 1.0, q_norm, 0, 1e-6, B, L, H, Hkv, D, 0)


@pytest.mark.parametrize("call,kw,code", [
    (_norm, dict(dtype=3), -4), (_norm, dict(odt=4), -4), (_norm, dict(K=0), -1), (_norm, dict(K=120), -1), (_norm, dict(K=124, odt=0), -1), (_norm, dict(K=32784), -2),
    (_norm, dict(pro=2), -3), (_norm, dict(pro=0), -3), (_norm, dict(pro=3, resid=0), -3), (_norm, dict(M=-1), -1), (_norm, dict(M=0), 0), (_norm, dict(x=0), -5), (_norm, dict(x=8), -5),
    (_norm, dict(xs=100), -5), (_norm, dict(xs=132), -5), (_norm, dict(resid=4), -5), (_norm, dict(resid_out=0), -5), (_norm, dict(ros=64), -5), (_norm, dict(w=8), -5),
    (_norm, dict(out=0), -5), (_norm, dict(os=136), -5), (_norm, dict(scales=0), -5), (_norm, dict(pro=3, resid=0, w=0, up=4), -5),
    (_linear, dict(odt=3), -4), (_linear, dict(K=24), -1), (_linear, dict(K=0), -1), (_linear, dict(K=32784), -2), (_linear, dict(beta=0.5), -207), (_linear, dict(M=-1), -1), (_linear, dict(M=0), 0),
    (_linear, dict(N=0), 0), (_linear, dict(x=8), -5), (_linear, dict(W=0), -5), (_linear, dict(x_stride=120), -5), (_linear, dict(x_stride=64), -5), (_linear, dict(out_stride=4), -5),
    (_linear, dict(xs=0), -5), (_linear, dict(M=2 ** 31 - 1), -1), (_linear, dict(N=2 ** 31 - 1), -1),
    (_requant, dict(dtype=3), -4), (_requant, dict(K=8), -1), (_requant, dict(N=-1), -1), (_requant, dict(N=0), 0), (_requant, dict(w=8), -5), (_requant, dict(stride=130), -5), (_requant, dict(codes=8), -5),
    (_requant, dict(N=2 ** 50), -1), (_requant, dict(N=2 ** 38), -1),
    (_dequant, dict(dtype=-1), -4), (_dequant, dict(rows=64), -1), (_dequant, dict(K=40), -1), (_dequant, dict(N=0), 0), (_dequant, dict(out=8), -5), (_dequant, dict(codes=0), -5), (_dequant, dict(N=2 ** 45), -1),
    (_packed, dict(dtype=0), -4), (_packed, dict(D=36), -1), (_packed, dict(D=264), -1), (_packed, dict(H=5), -1), (_packed, dict(Hkv=0), -1), (_packed, dict(B=0), 0), (_packed, dict(rows=0), 0),
    (_packed, dict(rows=-1), -1), (_packed, dict(q=8), -5), (_packed, dict(k=0), -5), (_packed, dict(offsets=0), -5), (_packed, dict(strides=odd), -5), (_packed, dict(strides=None), -5),
    (_packed, dict(rows=2 ** 31 - 1), -1), (_packed, dict(rows=2 ** 30, H=2 ** 20, Hkv=2 ** 20), -1), (_packed, dict(B=2 ** 31 - 1, H=64, Hkv=64), -1),
    (_rotary, dict(dtype=4), -4), (_rotary, dict(D=60, rot=60), -1), (_rotary, dict(D=264), -1), (_rotary, dict(rot=63), -1), (_rotary, dict(rot=66), -1), (_rotary, dict(L=0), 0), (_rotary, dict(B=-1), -1),
    (_rotary, dict(axes=0), -1), (_rotary, dict(axes=2), -5), (_rotary, dict(pos=0), -5), (_rotary, dict(freq=0), -5), (_rotary, dict(q=8), -5), (_rotary, dict(q_out=0), -5), (_rotary, dict(k=0), -5),
    (_rotary, dict(strides=odd), -5), (_rotary, dict(strides=None), -5), (_rotary, dict(q_norm=4), -5), (_rotary, dict(B=2 ** 31 - 1, L=2 ** 31 - 1), -1), (_rotary, dict(H=0, Hkv=0), 0)])
def test_codes(pkg, call, kw, code):
    assert call(pkg.lib, **kw) == code


@pytest.mark.parametrize("call,at", [(_packed, 6), (_packed, 7), (_rotary, 7), (_rotary, 8), (_rotary, 10), (_rotary, 11)])
def test_rows_of_the_result_in_one_place(pkg, call, at):
    strides = (C.c_int64 * 12)(*S)
    strides[at] = 0
    assert call(pkg.lib, strides=strides) == -5


def test_host_tensors_are_refused(pkg):
    A, L = pkg.attention, pkg.linear
    q, x = torch.zeros(4, 2, 64).half(), torch.zeros(4, 128)
    for call in (lambda: A.packed_attention(q, q, q, torch.zeros(2, dtype=torch.int32)), lambda: A.rotary(q[None], None, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(32).double()),
                 lambda: L.norm_rows(x), lambda: L.f8_requant(x), lambda: L.f8_dequant(x.to(torch.float8_e4m3fn), x), lambda: L.f8_linear(x.to(torch.float8_e4m3fn), x, x, x)):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()


def test_frequencies(pkg):
    f = pkg.attention.rope_frequencies
    plain, scale = f(128, device="cpu")
    assert plain.dtype == torch.float64 and scale == 1.0 and plain[0] == 1.0
    assert math.isclose(plain[63], 10000.0 ** (-126 / 128), rel_tol=1e-14)
    linear, scale = f(128, scaling="linear", factor=8.0, device="cpu")
    assert scale == 1.0 and torch.equal(linear, plain / 8)
    base, scale = f(128, scaling="base", factor=8.0, device="cpu")
    assert scale == 1.0 and base[0] == 1.0 and math.isclose(base[-1], plain[-1] / 8, rel_tol=1e-12) and bool((base <= plain).all())
    bands, scale = f(128, base=500000.0, scaling="bands", factor=16.0, trained=8192, device="cpu")
    plain, _ = f(128, base=500000.0, device="cpu")
    turns = 8192 * plain / (2 * math.pi)
    assert math.isclose(scale, 0.1 * math.log(16.0) + 1)
    assert torch.equal(bands[turns > 32], plain[turns > 32]) and torch.allclose(bands[turns < 1], plain[turns < 1] / 16, rtol=1e-15)
    assert bool((bands <= plain).all()) and bool((bands >= plain / 16 * (1 - 1e-15)).all())
    assert f(0, device="cpu")[0].shape == (0,) and f(2, scaling="base", factor=4.0, device="cpu")[0].tolist() == [1.0]
    for bad in (dict(rot=7), dict(rot=8, factor=0.5), dict(rot=8, scaling="other"), dict(rot=-2)):
        with pytest.raises(ValueError):
            f(**bad, device="cpu")
