"""The operators of the conditioning side of an engine -- linears with 4-bit weights and group scales, attention over a cache held
in 8 bits, cross attention to an encoder's states -- as cases with sizes: inputs, one pass, the bytes and operations that the pass
cannot do without.

``own = False`` computes a pass in its plain form, with elementary torch operations in 32 bits; ``own = True`` calls the library.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ---- the cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # Linears with 4-bit weights. One new token through the gate-up projection of a text encoder's MLP: latency and weight bytes.
        {"name": "w4_linear_m1", "op": "w4_linear", "M": 1, "K": 2560, "N": 19456, "G": 128, "dtype": "bf16", "zeros": False, "bias": False, "beta": 0},
        # The same MLP's down projection for a few tokens, f32 rows added to the residual stream, zero points, small groups, an odd N.
        {"name": "w4_linear_m5_f32", "op": "w4_linear", "M": 5, "K": 9728, "N": 2563, "G": 32, "dtype": "f32", "zeros": True, "bias": True, "beta": 1},
        # A whole prompt at once through a wide projection.
        {"name": "w4_linear_m333", "op": "w4_linear", "M": 333, "K": 5120, "N": 13824, "G": 64, "dtype": "f16", "zeros": False, "bias": True, "beta": 0},
        # A weight packed at load, and read back as a LoRA bake does.
        {"name": "w4_pack_bf16", "op": "w4_pack", "N": 13824, "K": 5120, "G": 128, "dtype": "bf16", "zeros": False},
        {"name": "w4_pack_f32_zeros", "op": "w4_pack", "N": 2563, "K": 9728, "G": 32, "dtype": "f32", "zeros": True},
        # The cache's writer: a new token of each of several sequences, and whole prompts of different lengths; then the rows read back.
        {"name": "kv8_store_token", "op": "kv8_store", "B": 8, "L": 1, "shortest": 40, "longest": 700, "Hkv": 8, "D": 128, "T": 64, "dtype": "bf16"},
        {"name": "kv8_store_prompts", "op": "kv8_store", "B": 4, "L": 777, "shortest": 0, "longest": 1029, "Hkv": 8, "D": 128, "T": 32, "dtype": "f16"},
        # Attention over the cache: one token of one conversation, one token each of a batch of long and short ones, a chunk of prompt.
        {"name": "kv8_attn_token", "op": "kv8_attn", "B": 1, "L": 1, "shortest": 1999, "longest": 1999, "H": 32, "Hkv": 8, "D": 128, "T": 64, "dtype": "bf16"},
        {"name": "kv8_attn_batch", "op": "kv8_attn", "B": 16, "L": 1, "shortest": 1, "longest": 32768, "H": 32, "Hkv": 8, "D": 128, "T": 64, "dtype": "f16"},
        {"name": "kv8_attn_chunk", "op": "kv8_attn", "B": 2, "L": 1024, "shortest": 1100, "longest": 4133, "H": 32, "Hkv": 8, "D": 128, "T": 32, "dtype": "bf16"},
        # Cross attention: the SDXL U-Net's 640-wide block at 1024 x 1024, CFG batch 2, prompts of 77 tokens, fp16.
        {"name": "cross_unet_640", "op": "cross", "B": 2, "Lq": 4096, "Lkv": 77, "H": 10, "Hkv": 10, "D": 64, "dtype": "f16", "lens": False, "mask": False},
        # A DiT at 2048 x 2048 that attends to a padded prompt of up to 512 tokens.
        {"name": "cross_dit_16384", "op": "cross", "B": 1, "Lq": 16384, "Lkv": 512, "H": 24, "Hkv": 24, "D": 128, "dtype": "bf16", "lens": False, "mask": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


_LARGEST = 4 * 24 * 16384 * 512 * 128          # multiply-adds times two of the largest listed case


def draw(rng):
    """One more case of the same ranges; no drawn case costs more than the largest listed one."""
    while True:
        case = _drawn(rng)
        # the plain form of attention holds a head's scores: what counts besides the products
        if work(case)["flops"] <= _LARGEST and work(case)["bytes"] <= 600e6:
            return case


def _drawn(rng):
    op = rng.choice(["w4_linear", "w4_linear", "w4_linear", "w4_pack", "kv8_store", "kv8_attn", "kv8_attn", "kv8_attn", "cross", "cross", "cross"])
    if op == "w4_linear":
        G = rng.choice([32, 64, 128])
        K = G * max(1, _log(rng, 256, 14336) // G)
        return {"op": op, "M": _log(rng, 1, 512) if rng.random() < 0.5 else rng.randint(1, 16), "K": K, "N": _log(rng, 64, 28672), "G": G,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "zeros": rng.random() < 0.5, "bias": rng.random() < 0.5, "beta": rng.randint(0, 1)}
    if op == "w4_pack":
        G = rng.choice([32, 64, 128])
        return {"op": op, "N": _log(rng, 200, 8192), "K": G * max(1, _log(rng, 512, 9728) // G), "G": G, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "zeros": rng.random() < 0.5}
    Hkv = rng.choice([1, 2, 4, 8, 16])
    if op == "kv8_store":
        L = rng.choice([1, 1, 2, 5, _log(rng, 8, 2048)])
        B = rng.randint(1, 16)
        low = rng.randint(0, 2000)
        return {"op": op, "B": B, "L": L, "shortest": low, "longest": low + rng.randint(0, 2000) + L, "Hkv": Hkv, "D": rng.choice([64, 80, 96, 128, 256]),
                "T": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "kv8_attn":
        L = rng.choice([1, 1, 1, 2, 4, _log(rng, 5, 1024)])
        low = _log(rng, 1, 16384)
        return {"op": op, "B": rng.randint(1, 24), "L": L, "shortest": low, "longest": max(low, _log(rng, 16, 40000)), "H": Hkv * rng.choice([1, 2, 3, 4, 8]),
                "Hkv": Hkv, "D": rng.choice([64, 80, 96, 128, 256]), "T": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "f16"])}
    H = rng.choice([5, 8, 10, 20, 24, 40])
    return {"op": op, "B": rng.choice([1, 1, 2, 3, 4]), "Lq": _log(rng, 1, 16384), "Lkv": _log(rng, 1, 2048), "H": H,
            "Hkv": H if rng.random() < 0.7 else H // rng.choice([d for d in (1, 2, 4, 5) if H % d == 0]), "D": rng.choice([40, 64, 80, 128, 160]),
            "dtype": rng.choice(["bf16", "f16"]), "lens": rng.random() < 0.5, "mask": rng.random() < 0.5}


def _lengths(case):
    """Keys of each sequence, spread evenly from the shortest to the longest (new ones included)."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    return [hi if B == 1 else lo + (hi - lo) * b // (B - 1) for b in range(B)]


def _new(case):
    """New tokens of each sequence: all L of them, or as many as it has."""
    return [min(case["L"], n) for n in _lengths(case)]


# ---- inputs ---------------------------------------------------------------------------------------------------------------

class _Make:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.dev)

    def activations(self, M, K):
        """N(0, 1) with heavy-tailed channels: a channel's scale is |t(3)|, between 0.2 and 50."""
        t = self.randn(K).abs() / (self.randn(3, K).square().sum(0) / 3.0).sqrt()
        return self.randn(M, K) * t.clamp(0.2, 50.0)

    def heads(self, *shape, spread=1.0):
        """Rows of queries or keys: N(0, 1) with channels of different scale, as projections without a norm leave them."""
        return self.randn(*shape) * (0.5 + self.randn(shape[-2], shape[-1]).abs() * spread)

    def ints(self, lo, hi, *shape, dtype=torch.uint8):
        return torch.randint(lo, hi, shape, generator=self.g, device=self.dev, dtype=torch.int32).to(dtype)


def _prepare_w4_linear(c, m):
    M, K, N, G, dt = c["M"], c["K"], c["N"], c["G"], _DT[c["dtype"]]
    s = {"x": m.activations(M, K).to(dt), "packed": m.ints(0, 256, N, K // 2), "G": G, "beta": c["beta"],
         "scales": (0.002 + 0.006 * torch.rand(N, K // G, generator=m.g, device=m.dev)).half()}
    s["zeros"] = m.ints(4, 12, N, K // G) if c["zeros"] else None
    s["bias"] = (m.randn(N) * 0.01).to(dt) if c["bias"] else None
    s["stream"] = m.activations(M, N).to(dt) if c["beta"] else None
    s["out"] = torch.empty((M, N), dtype=dt, device=m.dev)
    return s


def _prepare_w4_pack(c, m):
    return {"w": (m.randn(c["N"], c["K"]) * 0.02).to(_DT[c["dtype"]]), "G": c["G"], "zeros": c["zeros"]}


def _cache(c, m, lens):
    """A cache of pages in random order: codes, scales, the table, and a few pages that nobody uses."""
    B, T, Hkv, D = c["B"], c["T"], c["Hkv"], c["D"]
    width = max(lens) // T + 2 + (c["L"] - 1) // T
    used = B * width
    pages = used + 3
    order = torch.randperm(pages, generator=m.g, device=m.dev)[:used].to(torch.int32).view(B, width)
    return {"k8": m.ints(-127, 128, pages, Hkv, T, D, dtype=torch.int8), "v8": m.ints(-127, 128, pages, Hkv, T, D, dtype=torch.int8),
            "k_scale": 0.01 + 0.02 * torch.rand(pages, Hkv, generator=m.g, device=m.dev),
            "v_scale": 0.01 + 0.02 * torch.rand(pages, Hkv, generator=m.g, device=m.dev), "table": order.contiguous(),
            "lengths": torch.tensor(lens, dtype=torch.int32, device=m.dev)}


def _prepare_kv8_store(c, m):
    lens, new = _lengths(c), _new(c)
    s = _cache(c, m, lens)
    rows = m.heads(2, c["B"], c["L"], c["Hkv"], c["D"]).to(_DT[c["dtype"]])
    s.update(k=rows[0], v=rows[1], start=torch.tensor([n - a for n, a in zip(lens, new)], dtype=torch.int32, device=m.dev),
             count=torch.tensor(new, dtype=torch.int32, device=m.dev), longest=max(lens))
    return s


def _prepare_kv8_attn(c, m):
    lens, new = _lengths(c), _new(c)
    s = _cache(c, m, lens)
    q = m.heads(c["B"], c["L"], c["H"], c["D"]).to(_DT[c["dtype"]])
    s.update(q=q, out=torch.zeros_like(q), q_len=torch.tensor(new, dtype=torch.int32, device=m.dev) if min(new) < c["L"] else None)
    return s


def _prepare_cross(c, m):
    B, Lq, Lkv, H, Hkv, D, dt = c["B"], c["Lq"], c["Lkv"], c["H"], c["Hkv"], c["D"], _DT[c["dtype"]]
    s = {"q": m.heads(B, Lq, H, D).to(dt), "k": m.heads(B, Lkv, Hkv, D).to(dt), "v": m.randn(B, Lkv, Hkv, D).to(dt), "kv_len": None, "mask": None}
    if c["lens"]:
        s["kv_len"] = m.ints(0, Lkv + 1, B, dtype=torch.int32)
    if c["mask"]:           # a prompt's padding at its end, and single tokens struck out before it
        last = m.ints(max(1, Lkv // 2), Lkv + 1, B, 1, dtype=torch.int32)
        s["mask"] = (torch.arange(Lkv, device=m.dev) < last) & (torch.rand(B, Lkv, generator=m.g, device=m.dev) > 0.02)
    s["out"] = torch.empty_like(s["q"])
    return s


_PREPARE = {"w4_linear": _prepare_w4_linear, "w4_pack": _prepare_w4_pack, "kv8_store": _prepare_kv8_store, "kv8_attn": _prepare_kv8_attn,
            "cross": _prepare_cross}


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, _Make(seed))
    state["op"] = case["op"]
    if own:
        pkg = importlib.import_module("comfyui-backend-but-rust_b200")
        state["L"] = pkg.linear
        if case["op"].startswith("kv8"):
            state["A"] = pkg.attention
            state["cache"] = pkg.attention.Kv8Cache(state["k8"], state["v8"], state["k_scale"], state["v_scale"])
        elif case["op"] == "cross":
            state["A"] = pkg.attention
    return state


# ---- one pass: the library's calls ------------------------------------------------------------------------------------------

def _own_w4_linear(s):
    out = s["out"]
    if s["beta"]:
        out.copy_(s["stream"])          # the residual stream that the linear adds to
    return s["L"].w4_linear(s["x"], s["packed"], s["scales"], s["zeros"], s["bias"], out=out, beta=float(s["beta"]))


def _own_w4_pack(s):
    packed, scales, zeros = s["L"].w4_requant(s["w"], s["G"], zero_points=s["zeros"])
    return [s["L"].w4_dequant(packed, scales, zeros), scales]


def _own_kv8_store(s):
    s["A"].kv8_append(s["cache"], s["k"], s["v"], s["table"], s["start"], s["count"])
    return [*s["A"].kv8_dequant(s["cache"], s["table"], s["lengths"], s["longest"]), s["k_scale"], s["v_scale"]]


def _own_kv8_attn(s):
    return s["A"].kv8_attention(s["q"], s["cache"], s["table"], s["lengths"], q_len=s["q_len"], out=s["out"])


def _own_cross(s):
    return s["A"].cross_attention(s["q"], s["k"], s["v"], kv_len=s["kv_len"], key_mask=s["mask"], out=s["out"])


# ---- one pass: the plain form -----------------------------------------------------------------------------------------------

def _codes(packed):
    """Nibbles of [N, K / 2] bytes, the low one first, as [N, K]."""
    return torch.stack((packed & 15, packed >> 4), dim=2).flatten(1)


def _unpacked(packed, scales, zeros):
    N, groups = scales.shape
    z = 8.0 if zeros is None else zeros.float()[:, :, None]
    return ((_codes(packed).float().view(N, groups, -1) - z) * scales.float()[:, :, None]).view(N, -1)


def _plain_w4_linear(s):
    y = s["x"].float() @ _unpacked(s["packed"], s["scales"], s["zeros"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["beta"]:
        y = y + s["stream"].float()
    return y.to(s["x"].dtype)


def _plain_w4_pack(s):
    w = s["w"].float()
    g = w.view(w.shape[0], -1, s["G"])
    if s["zeros"]:
        lo, hi = g.amin(2).clamp_max(0.0), g.amax(2).clamp_min(0.0)
        scales = ((hi - lo) * (1.0 / 15.0)).half()
        st = scales.float()
        z = torch.where(st > 0, torch.round(-lo / st), 0.0).clamp(0, 15)[:, :, None]
    else:
        scales = (g.abs().amax(2) * (1.0 / 7.0)).half()
        st = scales.float()
        z = torch.full_like(st, 8.0)[:, :, None]
    st = st[:, :, None]
    codes = (torch.where(st > 0, torch.round(g / st), 0.0) + z).clamp(0, 15)
    return [((codes - z) * st).view_as(w), scales]


def _plain_written(codes, scale, rows, s):
    """One of K and V: new rows onto their pages, each page and head with one scale."""
    B, L, Hkv, D = rows.shape
    T = codes.shape[2]
    J = (L + T - 1) // T + 1
    dev = rows.device
    start, count = s["start"].long(), s["count"].long()
    first, off = start // T, start % T
    i = torch.arange(L, device=dev)
    at = off[:, None] + i                                                     # place on the pages from the first one touched
    fresh = (i < count[:, None])
    grid = torch.zeros((B, J * T, Hkv, D), device=dev)
    grid.scatter_(1, at[:, :, None, None].expand(B, L, Hkv, D), torch.where(fresh[:, :, None, None], rows.float(), 0.0))
    is_new = torch.zeros((B, J * T), dtype=torch.bool, device=dev).scatter_(1, at, fresh).view(B, J, 1, T, 1)
    grid = grid.view(B, J, T, Hkv, D).transpose(2, 3)
    page = s["table"].long().gather(1, first[:, None] + torch.arange(J, device=dev))
    before = (torch.arange(J * T, device=dev) < off[:, None]).view(B, J, 1, T, 1)   # rows that the first page held already
    old_codes, old_scale = codes[page], scale[page]
    touched, begun = is_new.any(3)[:, :, :, 0], before.any(3)[:, :, :, 0]
    new_scale = (grid.abs().amax((3, 4)) * (1.0 / 127.0)).clamp_min(1e-30)
    sc = torch.where(begun, torch.maximum(old_scale, new_scale), new_scale)
    q = torch.round(grid / sc[..., None, None]).clamp(-127, 127)
    kept = torch.round(old_codes.float() * (old_scale / sc)[..., None, None])
    out = torch.where(is_new, q, torch.where(before & touched[..., None, None], kept, old_codes.float()))
    codes[page] = out.to(torch.int8)
    scale[page] = torch.where(touched, sc, old_scale)


def _plain_rows(codes, scale, s, longest):
    """The rows of every sequence as [B, longest, Hkv, D]; zeros behind its last one."""
    B, (_, Hkv, T, D) = s["table"].shape[0], codes.shape
    page = s["table"][:, :(longest + T - 1) // T].long()
    rows = (codes[page].float() * scale[page][..., None, None]).transpose(2, 3).reshape(B, -1, Hkv, D)[:, :longest]
    seen = torch.arange(longest, device=codes.device) < s["lengths"][:, None]
    return torch.where(seen[:, :, None, None], rows, 0.0)


def _plain_kv8_store(s):
    out = []
    for codes, scale, rows in ((s["k8"], s["k_scale"], s["k"]), (s["v8"], s["v_scale"], s["v"])):
        _plain_written(codes, scale, rows, s)
        out.append(_plain_rows(codes, scale, s, s["longest"]))
    return [*out, s["k_scale"], s["v_scale"]]


def _plain_attention(q, k, v, seen, scale):
    """q [B, L, H, D], k and v [B, S, Hkv, D], seen [B, 1 or L, S]; a row that sees nothing is zeros."""
    B, L, H, D = q.shape
    Hkv = k.shape[2]
    q = q.float().view(B, L, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    p = (q @ k.float().permute(0, 2, 3, 1)).mul_(scale).view(B, Hkv, H // Hkv, L, -1)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    o = p.view(B, Hkv, -1, p.shape[-1]) @ v.float().transpose(1, 2)
    return o.view(B, Hkv, H // Hkv, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, H, D)


def _seen(s, longest):
    """Which keys each query sees: those up to its own position, the last query being the sequence's last token."""
    q_len = s["q_len"] if s["q_len"] is not None else torch.full_like(s["lengths"], s["q"].shape[1])
    at = (s["lengths"] - q_len)[:, None] + torch.arange(s["q"].shape[1], device=s["q"].device)
    return torch.arange(longest, device=s["q"].device) <= at[:, :, None]


def _plain_kv8_attn(s):
    q = s["q"]
    longest = s["table"].shape[1] * s["k8"].shape[2]
    k, v = (_plain_rows(s[c], s[f], s, longest) for c, f in (("k8", "k_scale"), ("v8", "v_scale")))
    y = _plain_attention(q, k, v, _seen(s, longest), q.shape[-1] ** -0.5).to(q.dtype)
    if s["q_len"] is None:
        return y
    live = torch.arange(q.shape[1], device=q.device) < s["q_len"][:, None]
    return torch.where(live[:, :, None, None], y, s["out"])          # rows behind a sequence's last query stay as they were


def _plain_cross(s):
    q, k = s["q"], s["k"]
    B, Lkv = k.shape[:2]
    seen = torch.ones((B, Lkv), dtype=torch.bool, device=q.device)
    if s["kv_len"] is not None:
        seen = seen & (torch.arange(Lkv, device=q.device) < s["kv_len"][:, None])
    if s["mask"] is not None:
        seen = seen & s["mask"]
    return _plain_attention(q, k, s["v"], seen[:, None], q.shape[-1] ** -0.5).to(q.dtype)


_PLAIN = {"w4_linear": _plain_w4_linear, "w4_pack": _plain_w4_pack, "kv8_store": _plain_kv8_store, "kv8_attn": _plain_kv8_attn, "cross": _plain_cross}
_OWN = {"w4_linear": _own_w4_linear, "w4_pack": _own_w4_pack, "kv8_store": _own_kv8_store, "kv8_attn": _own_kv8_attn, "cross": _own_cross}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _exact_softmax_rows(q, k, v, allowed):
    """One head of one sequence: q [L, D], k and v [S, D], allowed [L, S] or [S]."""
    z = torch.where(allowed, q @ k.t() / math.sqrt(q.shape[1]), -math.inf)
    w = torch.exp(z - z.amax(1, keepdim=True).nan_to_num(neginf=0.0))
    mass = w.sum(1, keepdim=True)
    return (w @ v) / torch.where(mass > 0, mass, 1.0)


def _exact_w4_linear(c, s):
    low, high = s["packed"].remainder(16), s["packed"].div(16, rounding_mode="floor")
    w = torch.empty((c["N"], c["K"]), dtype=torch.float64, device=low.device)
    w[:, 0::2], w[:, 1::2] = low.double(), high.double()
    z = s["zeros"].double() if c["zeros"] else torch.full_like(s["scales"], 8.0, dtype=torch.float64)
    w = (w - z.repeat_interleave(c["G"], 1)) * s["scales"].double().repeat_interleave(c["G"], 1)
    y = torch.einsum("mk,nk->mn", s["x"].double(), w)
    return y + (s["bias"].double() if c["bias"] else 0.0) + (s["stream"].double() if c["beta"] else 0.0)


def _exact_kv8_scales(c, s):
    T, out = c["T"], []
    for scale, rows in ((s["k_scale"], s["k"]), (s["v_scale"], s["v"])):
        now = scale.double()
        for b, (n, a) in enumerate(zip(_lengths(c), _new(c))):
            if a == 0:
                continue
            first = (n - a) // T
            at = torch.arange(n - a, n, device=now.device).div(T, rounding_mode="floor") - first
            top = torch.zeros((int((n - 1) // T - first + 1), c["Hkv"]), dtype=torch.float64, device=now.device)
            top.index_reduce_(0, at, rows[b, :a].double().abs().amax(2), "amax")
            page = s["table"][b, first:first + len(top)].long()
            top = (top / 127.0).clamp_min(1e-30)
            if (n - a) % T:                         # rows that the first page held already keep its scale from falling
                top[0] = torch.maximum(top[0], now[page[0]])
            now[page] = top
        out.append(now)
    return out


def _exact_kv8_attn(c, s):
    lens, new, T, ratio = _lengths(c), _new(c), c["T"], c["H"] // c["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, (n, a) in enumerate(zip(lens, new)):
        page = s["table"][b, :-(-n // T)].long()
        for h in range(c["Hkv"]):
            k, v = ((s[x][page, h].double() * s[f][page, h].double()[:, None, None]).flatten(0, 1)[:n] for x, f in (("k8", "k_scale"), ("v8", "v_scale")))
            allowed = torch.arange(n, device=k.device) <= torch.arange(n - a, n, device=k.device)[:, None]
            for j in range(h * ratio, (h + 1) * ratio):
                out[b, :a, j] = _exact_softmax_rows(s["q"][b, :a, j].double(), k, v, allowed)
    return out


def _exact_cross(c, s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    t = torch.arange(c["Lkv"], device=out.device)
    for b in range(c["B"]):
        allowed = t < (s["kv_len"][b] if c["lens"] else c["Lkv"])
        if c["mask"]:
            allowed = allowed & s["mask"][b]
        for h in range(c["H"]):
            g = h // (c["H"] // c["Hkv"])
            out[b, :, h] = _exact_softmax_rows(s["q"][b, :, h].double(), s["k"][b, :, g].double(), s["v"][b, :, g].double(), allowed)
    return out


def exact(case, seed):
    """Codes are decisions, not computed numbers: where an output is what they stand for there is None."""
    s = _PREPARE[case["op"]](case, _Make(seed))
    if case["op"] == "w4_pack":
        g = s["w"].double().unflatten(1, (-1, case["G"]))
        span = (g.amax(2).clamp(min=0) - g.amin(2).clamp(max=0)) / 15 if case["zeros"] else g.abs().amax(2) / 7
        return [None, span]
    if case["op"] == "kv8_store":
        return [None, None, *_exact_kv8_scales(case, s)]
    return {"w4_linear": _exact_w4_linear, "kv8_attn": _exact_kv8_attn, "cross": _exact_cross}[case["op"]](case, s)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    """Inputs and weights read once, results written once; two operations per multiply-add of the products. Packing and the cache's
    writer have no product: a division, a rounding and a comparison for each value."""
    c, op, e = case, case["op"], _SIZE[case["dtype"]]
    if op == "w4_linear":
        M, K, N = c["M"], c["K"], c["N"]
        weights = N * K // 2 + N * (K // c["G"]) * (3 if c["zeros"] else 2)
        return {"bytes": weights + e * M * K + e * M * N * (2 if c["beta"] else 1) + (e * N if c["bias"] else 0), "flops": 2 * M * N * K}
    if op == "w4_pack":         # read once, packed, and written back in f32 from the packed form
        N, K = c["N"], c["K"]
        packed = N * K // 2 + N * (K // c["G"]) * (3 if c["zeros"] else 2)
        return {"bytes": (e + 4) * N * K + 2 * packed, "flops": 5 * N * K}
    row = c["Hkv"] * c["D"]
    lens = _lengths(c) if "shortest" in c else None
    if op == "kv8_store":       # new rows in, their codes out, and every sequence's rows read back in f32
        new, B = sum(_new(c)), c["B"]
        return {"bytes": 2 * row * (new * (e + 1) + sum(lens) + 4 * B * max(lens)) + 8 * c["Hkv"] * sum(-(-n // c["T"]) for n in lens),
                "flops": 2 * row * (3 * new + sum(lens))}
    if op == "kv8_attn":
        pairs = sum(a * (n - a) + a * (a + 1) // 2 for n, a in zip(lens, _new(c)))
        return {"bytes": 2 * row * sum(lens) + 8 * c["Hkv"] * sum(-(-n // c["T"]) for n in lens) + 2 * e * sum(_new(c)) * c["H"] * c["D"],
                "flops": 4 * pairs * c["H"] * c["D"]}
    B, Lq, Lkv, H, D = c["B"], c["Lq"], c["Lkv"], c["H"], c["D"]
    return {"bytes": 2 * e * B * Lq * H * D + 2 * e * B * Lkv * row + (B * Lkv if c["mask"] else 0), "flops": 4 * B * Lq * Lkv * H * D}
