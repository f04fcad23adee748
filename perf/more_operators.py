"""The operators of a text encoder's layer between its cache and its 8-bit linears -- the residual's addition with the norm and the rows'
way into e4m3, the linear over e4m3 blocks, rotary positions, attention over packed prompts -- as cases with sizes: inputs, one pass,
the bytes and operations that the pass cannot do without.

``own = False`` computes a pass in its plain form, with elementary torch operations in 32 bits (angles in 64); ``own = True`` calls the
library.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_F8 = torch.float8_e4m3fn
_EPS = 1e-6


# ---- the cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One new token: its row added to the residual stream, normalised, as e4m3 for the next linear. Latency alone.
        {"name": "norm_token", "op": "norm", "M": 1, "K": 2560, "dtype": "bf16", "pro": "rms", "resid": True, "to": "e4m3"},
        # The MLP's gate and up halves of a prompt on their way into the down projection.
        {"name": "swiglu_m777", "op": "norm", "M": 777, "K": 9728, "dtype": "f16", "pro": "swiglu", "resid": False, "to": "e4m3"},
        # A DiT's rows at 2048 x 2048 with the text's behind them: the stream in f32, the norm's rows as 32-bit numbers again.
        {"name": "norm_m16896_f32", "op": "norm", "M": 16896, "K": 2560, "dtype": "f32", "pro": "rms", "resid": True, "to": "rows"},
        # One token through a text encoder's gate-up projection: the weight's bytes.
        {"name": "f8_linear_m1", "op": "f8_linear", "M": 1, "K": 2560, "N": 19456, "dtype": "bf16", "bias": False, "beta": 0},
        # A few tokens down again, f32 rows added to the residual stream, an odd number of outputs, a last block of 16 columns.
        {"name": "f8_linear_m7_f32", "op": "f8_linear", "M": 7, "K": 9744, "N": 2563, "dtype": "f32", "bias": True, "beta": 1},
        # A prompt through a wide projection, and a batch of prompts.
        {"name": "f8_linear_m333", "op": "f8_linear", "M": 333, "K": 5120, "N": 13824, "dtype": "f16", "bias": True, "beta": 0},
        {"name": "f8_linear_m4352", "op": "f8_linear", "M": 4352, "K": 5120, "N": 13824, "dtype": "bf16", "bias": False, "beta": 0},
        # Rotary positions: a token each of eight conversations, far along and scaled for it, heads normalised; a prompt whose heads turn in
        # part, neighbouring values as pairs; an image's rows with three axes of positions.
        {"name": "rotary_token", "op": "rotary", "B": 8, "L": 1, "H": 32, "Hkv": 8, "D": 128, "rot": 128, "interleaved": False, "norm": True, "axes": 1,
         "far": 120000, "scaling": "bands", "factor": 4.0, "dtype": "bf16"},
        {"name": "rotary_image", "op": "rotary", "B": 2, "L": 4179, "H": 24, "Hkv": 24, "D": 128, "rot": 96, "interleaved": True, "norm": False, "axes": 3,
         "far": 0, "scaling": "none", "factor": 1.0, "dtype": "f16"},
        # Attention over packed prompts: a batch of short ones as a U-Net's captions are, long and short ones together with an empty one and rows
        # behind the last, and one long conversation.
        {"name": "attn_captions", "op": "attn", "B": 16, "shortest": 5, "longest": 77, "behind": 0, "H": 12, "Hkv": 12, "D": 64, "causal": True, "dtype": "f16"},
        {"name": "attn_ragged", "op": "attn", "B": 6, "shortest": 0, "longest": 2049, "behind": 100, "H": 32, "Hkv": 8, "D": 128, "causal": True, "dtype": "bf16"},
        {"name": "attn_long", "op": "attn", "B": 1, "shortest": 8192, "longest": 8192, "behind": 0, "H": 32, "Hkv": 8, "D": 128, "causal": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


_LARGEST = 2 * 4352 * 5120 * 13824             # operations of the largest listed linear
_SCORES = 32 * 8192 * 8192                     # logits that the plain form of attention holds at once, of the largest listed case


def draw(rng):
    """One more case of the same ranges; no drawn case costs more than the largest listed one."""
    while True:
        case = _drawn(rng)
        w = work(case)
        if w["flops"] <= _LARGEST and w["bytes"] <= 700e6 and (case["op"] != "attn" or case["B"] * case["H"] * case["longest"] ** 2 <= _SCORES):
            return case


def _drawn(rng):
    op = rng.choice(["norm", "norm", "norm", "f8_linear", "f8_linear", "f8_linear", "f8_linear", "rotary", "rotary", "attn", "attn", "attn", "attn"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "norm":
        pro = rng.choice(["rms", "rms", "rms", "swiglu", "plain"])
        return {"op": op, "M": _log(rng, 1, 16896), "K": 16 * _log(rng, 8, 1024), "dtype": dtype, "pro": pro, "resid": pro == "rms" and rng.random() < 0.7,
                "to": "rows" if pro == "rms" and rng.random() < 0.3 else "e4m3"}
    if op == "f8_linear":
        return {"op": op, "M": rng.randint(1, 32) if rng.random() < 0.4 else _log(rng, 1, 4352), "K": 16 * _log(rng, 16, 864), "N": _log(rng, 64, 28672),
                "dtype": dtype, "bias": rng.random() < 0.5, "beta": rng.randint(0, 1)}
    if op == "rotary":
        D = rng.choice([64, 80, 96, 128, 256])
        Hkv = rng.choice([1, 2, 4, 8])
        L = rng.choice([1, 1, _log(rng, 2, 8192), _log(rng, 2, 8192)])
        scaling = rng.choice(["none", "linear", "bands"])
        return {"op": op, "B": rng.randint(1, 32 if L == 1 else 4), "L": L, "H": Hkv * rng.choice([1, 3, 4, 8]), "Hkv": Hkv, "D": D,
                "rot": rng.choice([D, D // 2, D // 16 * 8]), "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5, "axes": rng.choice([1, 1, 3]),
                "far": rng.choice([0, _log(rng, 100, 1000000)]), "scaling": scaling, "factor": 1.0 if scaling == "none" else float(rng.randint(2, 32)),
                "dtype": dtype}
    Hkv = rng.choice([1, 2, 4, 8, 12])
    B = rng.randint(1, 4) if rng.random() < 0.5 else rng.randint(5, 64)
    longest = _log(rng, 1, 8192 if B <= 4 else 1024)
    return {"op": op, "B": B, "shortest": longest if B == 1 else rng.randint(0, longest), "longest": longest, "behind": rng.choice([0, 0, rng.randint(1, 300)]),
            "H": Hkv * rng.choice([1, 1, 2, 3, 4, 5, 8]), "Hkv": Hkv, "D": rng.choice([64, 72, 80, 96, 128, 128]), "causal": rng.random() < 0.75,
            "dtype": rng.choice(["bf16", "f16"])}


def _lengths(case):
    """Rows of each sequence, spread evenly from the shortest to the longest and shuffled by a fixed rule."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    lens = [hi if B == 1 else lo + (hi - lo) * b // (B - 1) for b in range(B)]
    return [lens[(7 * b + 3) % B] for b in range(B)] if B % 7 else lens


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

    def heads(self, *shape):
        """Rows of queries or keys: N(0, 1) with channels of different scale, as projections without a norm leave them."""
        return self.randn(*shape) * (0.5 + self.randn(shape[-2], shape[-1]).abs())


def _blocks(x, rows):
    """x [M, K] padded with zeros to whole blocks of `rows` by 128, as [M / rows, rows, K / 128, 128]."""
    M, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % 128, 0, -M % rows))
    return x.view(-1, rows, x.shape[1] // 128, 128)


def _to_e4m3(x, rows):
    """Codes and scales of x [M, K] f32 with a scale for each block of `rows` by 128: s = amax / 448, code = x / s."""
    M, K = x.shape
    b = _blocks(x, rows)
    s = b.abs().amax((1, 3)).clamp_min(1e-30) * (1.0 / 448.0)
    codes = (b * s.reciprocal()[:, None, :, None]).clamp(-448.0, 448.0).to(_F8)
    return codes.view(-1, b.shape[2] * 128)[:M, :K].contiguous(), s


def _prepare_norm(c, m):
    M, K, dt = c["M"], c["K"], _DT[c["dtype"]]
    s = {"pro": c["pro"], "to": c["to"], "K": K}
    if c["pro"] == "swiglu":
        s["x"] = m.activations(M, 2 * K).clamp_(-30, 30).to(dt)
        return s
    s["x"] = m.activations(M, K).to(dt)
    if c["pro"] == "rms":
        s["w"] = 1.0 + 0.2 * m.randn(K)
    s["stream"] = s["stream_out"] = None
    if c["resid"]:
        s["stream"] = (m.activations(M, K) * 3.0).to(dt)
        s["stream_out"] = torch.empty_like(s["stream"])
    return s


def _prepare_f8_linear(c, m):
    M, K, N, dt = c["M"], c["K"], c["N"], _DT[c["dtype"]]
    x, xs = _to_e4m3(m.activations(M, K), 1)
    w, ws = _to_e4m3(m.randn(N, K) * (0.01 + 0.02 * torch.rand(N, 1, generator=m.g, device=m.dev)), 128)
    return {"x": x, "xs": xs, "w": w, "ws": ws, "bias": (m.randn(N) * 0.01).to(dt) if c["bias"] else None,
            "stream": m.activations(M, N).to(dt) if c["beta"] else None, "out": torch.empty((M, N), dtype=dt, device=m.dev)}


def _frequencies(c):
    """Radians a position for each pair, in 64 bits: 10000^(-2 i / rot); "linear": all of them divided by the factor; "bands": divided
    where a turn is longer than 4096 positions, kept where 32 turns fit into them, in proportion between."""
    half = c["rot"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    if c["scaling"] == "linear":
        f = f / c["factor"]
    if c["scaling"] == "bands":
        turns = 4096.0 * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        f = f / c["factor"] * (1 - keep) + f * keep
    return f


def _prepare_rotary(c, m):
    B, L, dt, A = c["B"], c["L"], _DT[c["dtype"]], c["axes"]
    q, k = m.heads(B, L, c["H"], c["D"]).to(dt), m.heads(B, L, c["Hkv"], c["D"]).to(dt)
    pos = c["far"] + torch.arange(L, device=m.dev).expand(B, L) + (torch.arange(B, device=m.dev) * 1013)[:, None]
    s = {"q": q, "k": k, "q_out": torch.empty_like(q), "k_out": torch.empty_like(k), "freq": _frequencies(c).to(m.dev),
         "interleaved": c["interleaved"], "q_norm": None, "k_norm": None, "axis": None, "scale": 1.0 if c["scaling"] != "bands" else 0.1 * math.log(c["factor"]) + 1.0}
    if A > 1:           # frame, row and column of an image 64 wide
        wide = 64
        pos = torch.stack((pos // (wide * wide), pos // wide % wide, pos % wide))
        s["axis"] = (torch.arange(c["rot"] // 2, device=m.dev) * A // (c["rot"] // 2)).to(torch.uint8)
    s["pos"] = pos.to(torch.int32).contiguous()
    if c["norm"]:
        s["q_norm"], s["k_norm"] = 1.0 + 0.2 * m.randn(c["D"]), 1.0 + 0.2 * m.randn(c["D"])
    return s


def _prepare_attn(c, m):
    lens, dt = _lengths(c), _DT[c["dtype"]]
    rows = sum(lens) + c["behind"]
    q, k = m.heads(rows, c["H"], c["D"]).to(dt), m.heads(rows, c["Hkv"], c["D"]).to(dt)
    offsets = torch.zeros(len(lens) + 1, dtype=torch.int32)
    offsets[1:] = torch.tensor(lens).cumsum(0)
    return {"q": q, "k": k, "v": m.randn(rows, c["Hkv"], c["D"]).to(dt), "offsets": offsets.to(m.dev), "causal": c["causal"], "longest": max(lens),
            "out": torch.full_like(q, 0.25)}


_PREPARE = {"norm": _prepare_norm, "f8_linear": _prepare_f8_linear, "rotary": _prepare_rotary, "attn": _prepare_attn}


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, _Make(seed))
    state["op"] = case["op"]
    return state


# ---- one pass: the library's calls ------------------------------------------------------------------------------------------

_modules = []


def _library():
    if not _modules:
        pkg = importlib.import_module("comfyui-backend-but-rust_b200")
        _modules.extend((pkg.linear, pkg.attention, pkg.ffi))
    return _modules


def _own_norm(s):
    L, _, F = _library()
    to = _F8 if s["to"] == "e4m3" else s["x"].dtype
    if s["pro"] == "swiglu":
        return L.norm_rows(s["x"], F.PRO_SWIGLU, K=s["K"], up_offset=s["K"], out_dtype=to)
    if s["pro"] == "plain":
        return L.norm_rows(s["x"], F.PRO_PLAIN, out_dtype=to)
    rows = L.norm_rows(s["x"], F.PRO_RMS, norm_w=s["w"], eps=_EPS, resid=s["stream"], resid_out=s["stream_out"], out_dtype=to)
    return [rows, s["stream_out"]]


def _own_f8_linear(s):
    out = s["out"]
    if s["stream"] is not None:
        out.copy_(s["stream"])          # the residual stream that the linear adds to
    return _library()[0].f8_linear(s["x"], s["xs"], s["w"], s["ws"], s["bias"], out=out, beta=0.0 if s["stream"] is None else 1.0)


def _own_rotary(s):
    return _library()[1].rotary(s["q"], s["k"], s["pos"], s["freq"], interleaved=s["interleaved"], axis=s["axis"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                                eps=_EPS, scale=s["scale"], q_out=s["q_out"], k_out=s["k_out"])


def _own_attn(s):
    return _library()[1].packed_attention(s["q"], s["k"], s["v"], s["offsets"], causal=s["causal"], out=s["out"])


# ---- one pass: the plain form -----------------------------------------------------------------------------------------------

def _plain_norm(s):
    x, K = s["x"], s["K"]
    stream = None
    if s["pro"] == "swiglu":
        gate = x[:, :K].float()
        y = gate * torch.sigmoid(gate) * x[:, K:].float()
    elif s["pro"] == "plain":
        y = x.float()
    else:
        if s["stream"] is not None:
            stream = s["stream_out"]
            stream.copy_((x.float() + s["stream"].float()).to(x.dtype))     # the norm is of the stream as it is kept
            x = stream
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + _EPS) * s["w"]
    rows = _to_e4m3(y, 1) if s["to"] == "e4m3" else y.to(x.dtype)
    return rows if s["pro"] != "rms" else [rows, stream]


def _values(codes, scales, rows):
    """What codes and the scales of blocks of `rows` by 128 stand for."""
    s = scales.repeat_interleave(rows, 0)[:codes.shape[0]].repeat_interleave(128, 1)[:, :codes.shape[1]]
    return codes.to(scales.dtype) * s


def _plain_f8_linear(s):
    y = _values(s["x"], s["xs"], 1) @ _values(s["w"], s["ws"], 128).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["stream"] is not None:
        y = y + s["stream"].float()
    return y.to(s["out"].dtype)


def _plain_turned(x, cos, sin, weight, interleaved):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS) * weight
    half = cos.shape[-1]
    turned = y[..., :2 * half]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    a, b = a * cos - b * sin, a * sin + b * cos
    both = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((both, y[..., 2 * half:]), -1).to(x.dtype)


def _plain_rotary(s):
    pos = s["pos"].double()
    place = pos[..., None] if s["axis"] is None else pos[s["axis"].long()].permute(1, 2, 0)
    angle = place * s["freq"]
    cos, sin = (angle.cos() * s["scale"]).float()[:, :, None], (angle.sin() * s["scale"]).float()[:, :, None]
    s["q_out"].copy_(_plain_turned(s["q"], cos, sin, s["q_norm"], s["interleaved"]))
    s["k_out"].copy_(_plain_turned(s["k"], cos, sin, s["k_norm"], s["interleaved"]))
    return [s["q_out"], s["k_out"]]


def _plain_attn(s):
    q, k, v, longest = s["q"], s["k"], s["v"], s["longest"]
    H, D, Hkv = q.shape[1], q.shape[2], k.shape[1]
    start, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    at = torch.arange(longest, device=q.device)
    there = at < (end - start)[:, None]                                     # [B, longest]
    row = torch.where(there, start[:, None] + at, 0)
    B = row.shape[0]
    qs = q[row].float().view(B, longest, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    ks, vs = k[row].float().permute(0, 2, 3, 1), v[row].float().transpose(1, 2)
    p = (qs @ ks).mul_(D ** -0.5).view(B, Hkv, H // Hkv, longest, longest)
    seen = there[:, None, :] & (at <= at[:, None]) if s["causal"] else there[:, None, :].expand(B, longest, longest)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    o = (p.view(B, Hkv, -1, longest) @ vs).view(B, Hkv, H // Hkv, longest, D).permute(0, 3, 1, 2, 4).reshape(B, longest, H, D)
    s["out"].index_copy_(0, row[there], o[there].to(q.dtype))               # rows behind the last sequence stay as they were
    return s["out"]


_OWN = {"norm": _own_norm, "f8_linear": _own_f8_linear, "rotary": _own_rotary, "attn": _own_attn}
_PLAIN = {"norm": _plain_norm, "f8_linear": _plain_f8_linear, "rotary": _plain_rotary, "attn": _plain_attn}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------------------

def _exact_norm(c, s):
    """The norm is of the stream in its type. Codes: the value over its scale, before its rounding to 8 bits."""
    K, dt = c["K"], _DT[c["dtype"]]
    x = s["x"].double()
    kept = None
    if c["pro"] == "swiglu":
        y = x[:, :K] / (1.0 + torch.exp(-x[:, :K])) * x[:, K:]
    elif c["pro"] == "plain":
        y = x
    else:
        if c["resid"]:
            kept = x + s["stream"].double()
            x = kept.to(dt).double()
        y = x / ((x * x).sum(1, keepdim=True) / K + _EPS).sqrt() * s["w"].double()
    if c["to"] == "e4m3":
        groups = -(-K // 128)
        wide = torch.zeros((y.shape[0], groups * 128), dtype=torch.float64, device=y.device)
        wide[:, :K] = y
        wide = wide.view(-1, groups, 128)
        scale = wide.abs().max(2).values.clamp_min(1e-30) / 448.0
        out = [(wide / scale[:, :, None]).reshape(y.shape[0], -1)[:, :K], scale]
    else:
        out = y
    return out if c["pro"] != "rms" else [out, kept]


def _exact_f8_linear(c, s):
    M, K, N = c["M"], c["K"], c["N"]
    y = torch.zeros((M, N), dtype=torch.float64, device=s["x"].device)
    of_row = torch.arange(N, device=y.device) // 128
    for g in range(-(-K // 128)):           # a block of columns at a time: its scales are of the sums
        a, b = s["x"][:, g * 128:(g + 1) * 128].double(), s["w"][:, g * 128:(g + 1) * 128].double()
        y += (a @ b.t()) * (s["xs"][:, g].double()[:, None] * s["ws"][:, g].double()[of_row])
    for extra in (s["bias"], s["stream"]):
        if extra is not None:
            y += extra.double()
    return y


def _exact_rotary(c, s):
    rot = c["rot"]
    out = []
    for x, weight in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        y = x.double()
        if weight is not None:
            y = y / ((y * y).sum(-1, keepdim=True) / c["D"] + _EPS).sqrt() * weight.double()
        z = y.clone()
        for i in range(rot // 2):
            axis = 0 if s["axis"] is None else int(s["axis"][i])
            place = (s["pos"] if s["axis"] is None else s["pos"][axis]).double()
            turn = torch.polar(torch.full_like(place, s["scale"]), place * s["freq"][i])[:, :, None]
            one, two = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)
            w = torch.complex(y[..., one], y[..., two]) * turn
            z[..., one], z[..., two] = w.real, w.imag
        out.append(z)
    return out


def _exact_attn(c, s):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    o = s["out"].double()
    at = 0
    for n in _lengths(c):
        for h in range(H):
            if n == 0:
                break
            k, v = s["k"][at:at + n, h // (H // Hkv)].double(), s["v"][at:at + n, h // (H // Hkv)].double()
            logits = s["q"][at:at + n, h].double() @ k.t() / math.sqrt(D)
            if c["causal"]:
                logits = logits + torch.full_like(logits, -math.inf).triu(1)
            o[at:at + n, h] = torch.softmax(logits, 1) @ v
        at += n
    return o


def exact(case, seed):
    state = _PREPARE[case["op"]](case, _Make(seed))
    return {"norm": _exact_norm, "f8_linear": _exact_f8_linear, "rotary": _exact_rotary, "attn": _exact_attn}[case["op"]](case, state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    """Inputs and weights read once, results written once; two operations per multiply-add of the products. Norms and rotations: a few
    operations for each value."""
    c, op, e = case, case["op"], _SIZE[case["dtype"]]
    if op == "norm":
        M, K = c["M"], c["K"]
        rows = e * M * K * (2 if c["pro"] == "swiglu" else 3 if c["resid"] else 1)
        out = M * K + 4 * M * -(-K // 128) if c["to"] == "e4m3" else e * M * K
        return {"bytes": rows + out + (4 * K if c["pro"] == "rms" else 0), "flops": 6 * M * K}
    if op == "f8_linear":
        M, K, N = c["M"], c["K"], c["N"]
        scales = 4 * -(-K // 128) * (M + -(-N // 128))
        return {"bytes": N * K + M * K + scales + e * M * N * (2 if c["beta"] else 1) + (e * N if c["bias"] else 0), "flops": 2 * M * N * K}
    if op == "rotary":
        rows, heads = c["B"] * c["L"], c["H"] + c["Hkv"]
        return {"bytes": 2 * e * rows * heads * c["D"] + 4 * rows * c["axes"], "flops": rows * heads * (3 * c["rot"] + (4 * c["D"] if c["norm"] else 0))}
    lens = _lengths(c)
    pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lens)
    return {"bytes": 2 * e * sum(lens) * c["D"] * (c["H"] + c["Hkv"]), "flops": 4 * pairs * c["H"] * c["D"]}
