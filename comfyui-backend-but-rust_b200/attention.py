"""Host side of the attention that stands between the quantized linears, over torch CUDA tensors: cross attention to an encoder's
states (a U-Net's or DiT's image rows over a prompt's), and the cache of int8 keys and values that a text encoder's or a video
model's steps fill and attend to. torch supplies device memory and the stream only.

Every call runs on the device of its tensors, on that device's current stream.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .linear import _h


def _scale(q: torch.Tensor, scale: Optional[float]) -> float:
    return scale if scale is not None else max(q.shape[-1], 1) ** -0.5


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_len: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gpu_cross_attention: softmax(scale q k^T) v. q [B, Lq, H, D], k and v [B, Lkv, Hkv, D], fp16 or bf16, any strides of whole
    16-byte pieces; D a multiple of 8 up to 256; H a multiple of Hkv (head h reads kv head h // (H // Hkv)). Keys from kv_len[b]
    (int32 [B]) on, and those whose key_mask (bool [B, Lkv]) is False, are not seen, whatever they hold; a query that sees none gets
    zeros. `scale` defaults to D ** -0.5. `out` may be q itself."""
    return _h.cross_attention(q, k, v, kv_len, key_mask, _scale(q, scale), out)


@dataclass
class Kv8Cache:
    """Keys and values in 8 bits: k, v int8 [pages, Hkv, T, D] and k_scale, v_scale f32 [pages, Hkv]; a value is code * scale. A page
    holds T = 16, 32, 64 or 128 tokens; D is a multiple of 16 up to 256. Which pages a sequence has, in order, is its row of a table
    int32 [B, pages to a sequence] that the caller keeps."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @staticmethod
    def empty(pages: int, heads: int, D: int, T: int = 64, device="cuda") -> "Kv8Cache":
        def zeros(*shape, dtype):
            return torch.zeros(shape, dtype=dtype, device=device)
        return Kv8Cache(zeros(pages, heads, T, D, dtype=torch.int8), zeros(pages, heads, T, D, dtype=torch.int8),
                        zeros(pages, heads, dtype=torch.float32), zeros(pages, heads, dtype=torch.float32))


def kv8_append(cache: Kv8Cache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
               count: Optional[torch.Tensor] = None) -> Kv8Cache:
    """gpu_kv8_append: rows k[b, i], v[b, i] ([B, L, Hkv, D], f32 / f16 / bf16) become tokens start[b] + i of sequence b, for i < count[b]
    (int32 [B]; all L without). A page that a sequence writes belongs to it alone, and to one
    entry of its table. Rows that fall on no page are dropped."""
    _h.kv8_append(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, table, start, count)
    return cache


def kv8_dequant(cache: Kv8Cache, table: torch.Tensor, lengths: torch.Tensor, rows: int, *, dtype=torch.float32):
    """gpu_kv8_dequant: (k, v) [B, rows, Hkv, D] of the sequences' first `rows` tokens; zeros from lengths[b] on."""
    return _h.kv8_dequant(cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths, rows, dtype)


def kv8_attention(q: torch.Tensor, cache: Kv8Cache, table: torch.Tensor, lengths: torch.Tensor, *, q_len: Optional[torch.Tensor] = None,
                  causal: bool = True, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gpu_kv8_attention: softmax(scale q k^T) v over the first lengths[b] tokens of each sequence. q [B, L, H, D] fp16 or bf16, H a
    multiple of the cache's heads. The first q_len[b] (all L without) rows of q are the sequence's last tokens: causal, row i sees
    tokens up to lengths[b] - q_len[b] + i. Rows from q_len[b] on are not written; a row that sees no token gets zeros. `out`
    may be q itself."""
    return _h.kv8_attention(cache.k, cache.v, cache.k_scale, cache.v_scale, q, table, lengths, q_len, 1 if causal else 0,
                            _scale(q, scale), out)
