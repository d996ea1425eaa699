"""The operators around an attention layer's 4-bit cache as programs call them: the norm of each query's
and key's head with the position rotation in the same pass (one axis of positions for text, three for the
voxels of a volume), tokens written to the cache and read back, a cache's tokens read in 16 or 32 bits,
and the attention that reads the cache as it is.

4-bit values are OCP e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times a power of two held
in one byte (E8M0, ``2^(b - 127)``) for each 32 channels of a token: the least with which the block's
largest magnitude does not pass 6, and 1 for a block of zeros.
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

_PKG = "lesiondiffusion-mlx_amd"
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
_BLOCK = 32   # channels of a token that share a scale
_PAGE = 64    # tokens of a cache page
_EPS = 1e-6
_THETA = 10000.0
_HELD = 0.5 + 1 / _BLOCK   # bytes of a value in the cache


def listed() -> list[dict]:
    return [
        # One new token of a text's sequence, far along it: the smallest call, where the launch and the host count.
        {"name": "rotate_token", "kind": "rotate", "dtype": "fp16", "b": 1, "l": 1, "heads": 8, "kv": 8, "d": 64,
         "axes": "64", "interleaved": False, "norm": True, "first": 100_000},
        # The 51,200 voxels of a latent volume, 16 heads of 32: positions in three axes.
        {"name": "rotate_volume", "kind": "rotate", "dtype": "fp16", "b": 1, "l": 51200, "heads": 16, "kv": 16, "d": 32,
         "axes": "8,12,12", "interleaved": False, "norm": True, "first": 0},
        # Two volumes of an odd number of voxels in 32 bits, neighbouring channels turned, without norms.
        {"name": "rotate_odd", "kind": "rotate", "dtype": "fp32", "b": 2, "l": 1601, "heads": 5, "kv": 5, "d": 80,
         "axes": "16,30,30", "interleaved": True, "norm": False, "first": 0},
        # A long prompt's queries and shared keys: the largest pass of memory.
        {"name": "rotate_prompt", "kind": "rotate", "dtype": "bf16", "b": 1, "l": 16384, "heads": 32, "kv": 8, "d": 128,
         "axes": "128", "interleaved": False, "norm": True, "first": 30_000},
        # One new token for each of 48 sequences of unequal lengths, written and read back as it is held.
        {"name": "store_tokens", "kind": "store", "dtype": "bf16", "b": 48, "heads": 8, "d": 128, "n": 1, "held": 2000},
        # A prompt of an odd length behind held tokens; its own attention goes by what the cache holds.
        {"name": "store_prompt", "kind": "store", "dtype": "fp16", "b": 2, "heads": 8, "d": 64, "n": 4001, "held": 100},
        # A short sequence read into the type that another attention takes.
        {"name": "read_short", "kind": "read", "dtype": "fp16", "b": 1, "heads": 8, "d": 64, "held": 300},
        # Long sequences moved out of the cache.
        {"name": "read_long", "kind": "read", "dtype": "bf16", "b": 4, "heads": 8, "d": 128, "held": 24000},
        # One sequence, one query, a few pages: the smallest attention call.
        {"name": "attend_token", "kind": "attend", "dtype": "fp16", "b": 1, "heads": 8, "group": 1, "d": 64, "lq": 1,
         "held": 300, "causal": False},
        # One step of 32 sequences of unequal lengths with grouped heads: the cache's bytes decide.
        {"name": "attend_batch", "kind": "attend", "dtype": "bf16", "b": 32, "heads": 8, "group": 4, "d": 128, "lq": 1,
         "held": 16384, "causal": True},
        # One long sequence: few rows, so the tokens are what can be spread over the card.
        {"name": "attend_long", "kind": "attend", "dtype": "fp16", "b": 1, "heads": 4, "group": 8, "d": 128, "lq": 1,
         "held": 200_000, "causal": False},
        # A prompt's part of 2,000 queries behind held tokens, causal: bound by the matrix units.
        {"name": "attend_prompt", "kind": "attend", "dtype": "fp16", "b": 1, "heads": 4, "group": 4, "d": 64,
         "lq": 2000, "held": 8000, "causal": True},
    ]


# ------------------------------------------------------------------ drawn cases

def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _axes(rng, d: int) -> str:
    """One to three even widths that take all of ``d`` channels or leave some of them as they are."""
    n = rng.choice([1, 1, 2, 3, 3])
    whole = d if rng.random() < 0.7 else max(2 * n, d // 4 * 2)
    if n == 1:
        return str(whole)
    each = max(2, whole // n // 2 * 2)
    return ",".join(str(w) for w in [whole - (n - 1) * each] + [each] * (n - 1))


def draw(rng) -> dict:
    kind = rng.choice(["rotate", "rotate", "store", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
    if kind == "rotate":
        d = rng.choice([32, 48, 64, 64, 72, 80, 96, 128, 128, 160, 256])
        b, kv = _log(rng, 1, 16), rng.choice([1, 2, 4, 5, 8, 16])
        heads = kv * rng.choice([1, 1, 2, 4])
        l = _log(rng, 1, max(2, min(60_000, 80_000_000 // (b * (heads + kv) * d))))
        return {"kind": kind, "dtype": dtype, "b": b, "l": l, "heads": heads, "kv": kv, "d": d, "axes": _axes(rng, d),
                "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.7, "first": rng.choice([0, _log(rng, 1, 500_000)])}
    d = rng.choice([32, 64, 64, 128, 128, 256])
    heads = rng.choice([1, 2, 4, 5, 8, 16])
    if kind == "store":
        b = _log(rng, 1, 64)
        n = rng.choice([1, 1, _log(rng, 2, 8192)])
        n = max(1, min(n, 30_000_000 // (b * heads * d)))
        held = _log(rng, 1, max(2, min(4096, 60_000_000 // (b * heads * d))))
        return {"kind": kind, "dtype": dtype, "b": b, "heads": heads, "d": d, "n": n, "held": held}
    if kind == "read":
        b = _log(rng, 1, 32)
        held = _log(rng, 1, max(2, min(60_000, 60_000_000 // (b * heads * d))))
        return {"kind": kind, "dtype": dtype, "b": b, "heads": heads, "d": d, "held": held}
    dtype = rng.choice(["fp16", "bf16"])
    group = rng.choice([1, 1, 2, 4, 8])
    if rng.random() < 0.65:
        b, lq = _log(rng, 1, 64), rng.choice([1, 1, 1, rng.randint(2, 8)])
        held = _log(rng, 1, max(2, min(200_000, 260_000_000 // (b * heads * d))))
        return {"kind": kind, "dtype": dtype, "b": b, "heads": heads, "group": group, "d": d, "lq": lq, "held": held,
                "causal": rng.random() < 0.7}
    b, lq = rng.choice([1, 1, 2, 3]), _log(rng, 9, 4096)
    held = _log(rng, 16, 8192)
    lq = max(9, min(lq, 250_000_000 // (b * heads * group * (held + lq))))
    return {"kind": kind, "dtype": dtype, "b": b, "heads": heads, "group": group, "d": d, "lq": lq, "held": held,
            "causal": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs

def _held(case: dict) -> list[int]:
    """Tokens held for each sequence before the call: from ``held`` down to a quarter of it."""
    b, most = case["b"], case["held"]
    return [max(1, most - (i * 5 % b) * 3 * most // (4 * b)) for i in range(b)]


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _widths(case: dict) -> list[int]:
    return [int(w) for w in case["axes"].split(",")]


def _grid(l: int, axes: int) -> list[int]:
    """Extents of a volume (or plane) that holds ``l`` places."""
    side = max(1, round(l ** (1 / axes)))
    return [max(1, -(-l // side ** (axes - 1)))] + [side] * (axes - 1)


def _positions(case: dict, g: torch.Generator) -> torch.Tensor:
    """int32 (axes, B, L): a text's from ``first`` on, a part of a volume's in its order for several axes."""
    axes, b, l = len(_widths(case)), case["b"], case["l"]
    at = torch.arange(l, device="cuda").expand(b, l)
    if axes == 1:
        first = case["first"] + torch.randint(0, 1000, (b, 1), generator=g, device="cuda")
        return (at + first)[None].to(torch.int32)
    grid, out = _grid(l, axes), []
    for a in range(axes):
        inner = math.prod(grid[a + 1:])
        out.append(at // inner % grid[a] + case["first"])
    return torch.stack(out).to(torch.int32)


def _exponent(amax: torch.Tensor) -> torch.Tensor:
    """The scale byte of blocks whose largest magnitude is ``amax`` (fp32), as int32."""
    bits = amax.view(torch.int32)
    e = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000).to(torch.int32)).clamp(min=1)
    return torch.where(amax > 0, e, 127)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^(e - 127) in fp32 for int32 ``e`` of 1 to 254."""
    return (e << 23).view(torch.float32)


def _rows4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(..., D) as packed codes (..., D / 2), the even channel in the lower four bits, and scale bytes (..., D / 32)."""
    y = x.float().unflatten(-1, (-1, _BLOCK))
    e = _exponent(y.abs().amax(-1))
    y = (y * _pow2(254 - e)[..., None]).flatten(-2)
    m = y.abs()
    code = (m > 0.25).to(torch.uint8)
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (m >= border if up else m > border).to(torch.uint8)   # ties to the even code
    code |= torch.signbit(y).to(torch.uint8) << 3
    return code[..., 0::2] | code[..., 1::2] << 4, e.to(torch.uint8)


def _codes(device) -> torch.Tensor:
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)
    return torch.cat([v, -v])


def _wide(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 (..., D) of packed codes (..., D / 2) and scale bytes (..., D / 32)."""
    of = _codes(codes.device)
    v = torch.stack([of[(codes & 15).int()], of[(codes >> 4).int()]], -1).flatten(-2)
    return (v.unflatten(-1, (-1, _BLOCK)) * _pow2(scales.int())[..., None]).flatten(-2)


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    t = _DTYPES[case["dtype"]]
    st = dict(case)
    d = case["d"]
    if case["kind"] == "rotate":
        b, l, heads, kv = case["b"], case["l"], case["heads"], case["kv"]
        # What the projection of queries, keys and values wrote: heads differ in size.
        loud = 0.5 + 3 * torch.rand(heads + 2 * kv, 1, generator=g, device="cuda")
        qkv = torch.randn(b, l, heads + 2 * kv, d, generator=g, device="cuda").mul_(loud).to(t)
        st["q"], st["k"] = qkv[:, :, :heads].transpose(1, 2), qkv[:, :, heads:heads + kv].transpose(1, 2)
        st["positions"] = _positions(case, g)
        st["q_gamma"], st["k_gamma"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None
                                        for _ in range(2))
        # The table that a program makes once: turns per position of every pair of channels, axis by axis.
        st["turns"] = torch.cat([torch.pow(_THETA, -2.0 * torch.arange(w // 2, dtype=torch.float64, device="cuda") / w)
                                 for w in _widths(case)]) / (2 * math.pi)
        return st
    b, h, held = case["b"], case["heads"], _held(case)
    new = {"store": case.get("n"), "read": 0, "attend": case.get("lq")}[case["kind"]]
    width = -(-(max(held) + new) // _PAGE)
    pages = b * width + 1   # the last page is in no table
    loud = 1 + 3 * torch.rand(h, 1, d, generator=g, device="cuda")
    for name, size in (("k", loud), ("v", 1.0)):
        x = torch.randn(pages, h, _PAGE, d, generator=g, device="cuda") * size
        codes, scales = zip(*(_rows4(part) for part in x.split(max(1, (1 << 24) // (h * _PAGE * d)))))
        st[name + "_codes"] = torch.cat(codes)
        st[name + "_scales"] = torch.cat(scales).transpose(2, 3).contiguous()
        del x, codes, scales
    st["table"] = torch.randperm(pages - 1, generator=g, device="cuda").to(torch.int32).reshape(b, width)
    st["starts"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    st["lengths"] = st["starts"] + new
    if case["kind"] == "store":
        st["k"] = (torch.randn(b, h, new, d, generator=g, device="cuda") * 1.5 * loud).to(t)
        st["v"] = (torch.randn(b, h, new, d, generator=g, device="cuda") * 1.5).to(t)
    elif case["kind"] == "attend":
        st["q"] = torch.randn(b, h * case["group"], new, d, generator=g, device="cuda").to(t)
    return st


# ------------------------------------------------------------------ plain forms

def _pairs(case: dict, device) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """For every turned pair of channels: its first and second channel and its axis."""
    first, second, axis, at = [], [], [], 0
    for a, w in enumerate(_widths(case)):
        i = torch.arange(w // 2, device=device)
        first.append(at + (2 * i if case["interleaved"] else i))
        second.append(first[-1] + (1 if case["interleaved"] else w // 2))
        axis.append(torch.full_like(i, a))
        at += w
    return torch.cat(first), torch.cat(second), torch.cat(axis)


def _turned(x: torch.Tensor, gamma: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, first: torch.Tensor,
            second: torch.Tensor) -> torch.Tensor:
    f = x.float()
    if gamma is not None:
        f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS) * gamma
    y = f.clone()
    a, b = f[..., first], f[..., second]
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    return y.to(x.dtype)


def _rotate(st: dict) -> dict:
    first, second, axis = _pairs(st, st["q"].device)
    at = st["positions"].double()[axis].permute(1, 2, 0) * st["turns"]      # (B, L, pairs)
    angle = (at - torch.floor(at)) * (2 * math.pi)                          # far positions lose their angle in 32 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    return {"q": _turned(st["q"], st["q_gamma"], cos, sin, first, second),
            "k": _turned(st["k"], st["k_gamma"], cos, sin, first, second)}


def _places(st: dict, first: torch.Tensor, n: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Page and place in it of tokens first .. first + n of every sequence, (B, n) each."""
    pos = first.long()[:, None] + torch.arange(n, device=first.device)
    return st["table"].long().gather(1, pos // _PAGE), pos % _PAGE


def _store(st: dict) -> dict:
    page, slot = _places(st, st["starts"], st["n"])
    out = {}
    for name in ("k", "v"):
        codes, scales = _rows4(st[name].transpose(1, 2))                    # (B, n, H, ..)
        st[name + "_codes"][page, :, slot] = codes
        st[name + "_scales"][page, :, :, slot] = scales
        out[name] = _wide(st[name + "_codes"][page, :, slot], st[name + "_scales"][page, :, :, slot]) \
            .transpose(1, 2).to(st[name].dtype)
    return out


def _read(st: dict) -> dict:
    n, t = st["held"], _DTYPES[st["dtype"]]
    page, slot = _places(st, torch.zeros_like(st["starts"]), n)
    within = (torch.arange(n, device=page.device) < st["lengths"][:, None])[:, None, :, None]
    out = {}
    for name in ("k", "v"):
        x = _wide(st[name + "_codes"][page, :, slot], st[name + "_scales"][page, :, :, slot])
        out[name] = torch.where(within, x.transpose(1, 2), 0.0).to(t)
    return out


def _attend(st: dict) -> torch.Tensor:
    q, table, scale = st["q"], st["table"].long(), st["d"] ** -0.5
    b, hq, lq, d = q.shape
    h, n = st["heads"], table.shape[1] * _PAGE
    k = _wide(st["k_codes"][table], st["k_scales"][table].transpose(3, 4))                # (B, W, H, 64, D)
    k = k.permute(0, 2, 4, 1, 3).reshape(b, h, d, n)
    s = torch.matmul(q.float().reshape(b, h, hq // h * lq, d), k).reshape(b, h, hq // h, lq, n) * scale
    del k
    key = torch.arange(n, device=q.device)
    seen = key < st["lengths"][:, None, None]
    if st["causal"]:
        seen = seen & (key <= st["starts"][:, None, None] + torch.arange(lq, device=q.device)[:, None])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(4, keepdim=True))
    v = _wide(st["v_codes"][table], st["v_scales"][table].transpose(3, 4))
    v = v.permute(0, 2, 1, 3, 4).reshape(b, h, n, d)
    o = torch.matmul(p.reshape(b, h, hq // h * lq, n), v).reshape(b, h, hq // h, lq, d) / p.sum(4, keepdim=True)
    return o.reshape(b, hq, lq, d).to(q.dtype)


def run(st: dict):
    kind = st["kind"]
    if not own:
        return {"rotate": _rotate, "store": _store, "read": _read, "attend": _attend}[kind](st)
    ops = importlib.import_module(_PKG).ops
    if kind == "rotate":
        rotary = ops.Rotary(st["turns"], tuple(_widths(st)), st["interleaved"])
        q, k = ops.rotate_heads(st["q"], st["k"], st["positions"], rotary, q_gamma=st["q_gamma"],
                                k_gamma=st["k_gamma"], eps=_EPS)
        return {"q": q, "k": k}
    e8m0 = torch.float8_e8m0fnu
    cache = ops.Cache4(st["k_codes"], st["v_codes"], st["k_scales"].view(e8m0), st["v_scales"].view(e8m0))
    if kind == "store":
        ops.cache4_append(cache, st["k"], st["v"], st["table"], st["starts"])
        k, v = ops.cache4_read(cache, st["table"], st["lengths"], st["n"], starts=st["starts"], dtype=st["k"].dtype)
        return {"k": k, "v": v}
    if kind == "read":
        k, v = ops.cache4_read(cache, st["table"], st["lengths"], st["held"], dtype=_DTYPES[st["dtype"]])
        return {"k": k, "v": v}
    return ops.cache4_attention(st["q"], cache, st["table"], st["lengths"], st["d"] ** -0.5,
                                starts=st["starts"] if st["causal"] else None)


# ------------------------------------------------------------------ the work itself

def _visible(case: dict) -> int:
    """(query, key) pairs of one head, over all sequences."""
    lq, total = case["lq"], 0
    for n in _held(case):
        total += lq * n + (lq * (lq + 1) // 2 if case["causal"] else lq * lq)
    return total


def work(case: dict) -> dict:
    size, d, b = _BYTES[case["dtype"]], case["d"], case["b"]
    if case["kind"] == "rotate":
        places = b * case["l"]
        n = places * (case["heads"] + case["kv"]) * d
        return {"bytes": 2 * n * size + 4 * places * len(_widths(case)), "flops": (7 if case["norm"] else 3) * n}
    h = case["heads"]
    if case["kind"] == "store":
        n = b * h * case["n"] * d
        return {"bytes": 2 * n * (2 * size + _HELD), "flops": 6 * n}
    if case["kind"] == "read":
        held = sum(_held(case)) * h * d
        return {"bytes": 2 * held * _HELD + 2 * b * h * case["held"] * d * size, "flops": 2 * held}
    keys = sum(_held(case)) + b * case["lq"]
    rows = b * h * case["group"] * case["lq"]
    return {"bytes": 2 * keys * h * d * _HELD + 2 * rows * d * size,
            "flops": 4 * h * case["group"] * d * _visible(case)}


# ------------------------------------------------------------------ 64-bit results

def _exact_rotate(st: dict) -> dict:
    """Each pair as a complex number, multiplied by exp(i * angle)."""
    out = {}
    for name in ("q", "k"):
        x, gamma = st[name].double(), st[name + "_gamma"]
        if gamma is not None:
            x = x / torch.sqrt(x.pow(2).sum(3, keepdim=True) / st["d"] + _EPS) * gamma.double()
        parts, at = [], 0
        for a, w in enumerate(_widths(st)):
            part, half = x[..., at:at + w], w // 2
            freq = torch.tensor([_THETA ** (-2.0 * i / w) for i in range(half)], dtype=torch.float64, device=x.device)
            z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), st["positions"][a].double()[:, None, :, None] * freq)
            if st["interleaved"]:
                y = torch.complex(part[..., 0::2], part[..., 1::2]) * z
                parts.append(torch.stack([y.real, y.imag], 4).reshape(part.shape))
            else:
                y = torch.complex(part[..., :half], part[..., half:]) * z
                parts += [y.real, y.imag]
            at += w
        out[name] = torch.cat(parts + [x[..., at:]], 3)
    return out


def _nearest4(x: torch.Tensor) -> torch.Tensor:
    """float64 (..., D) as the nearest 4-bit values under each block's scale, ties to the even code."""
    y = x.unflatten(-1, (-1, _BLOCK))
    amax = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.clamp(amax, min=1e-300) / 6.0)).clamp(min=-126)
    e = torch.where(6.0 * torch.exp2(e - 1) >= amax, e - 1, e).clamp(min=-126)
    e = torch.where(6.0 * torch.exp2(e) < amax, e + 1, e)
    y = y / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)   # 0.5 below 2, 1 below 4, 2 from there
    return (torch.round(y / step) * step * torch.exp2(e)).flatten(-2)


def _tokens(st: dict, name: str, i: int, n: int) -> torch.Tensor:
    """float64 (H, n, D): what the cache holds of sequence i's first n tokens."""
    at = st["table"][i, :-(-n // _PAGE)].long()
    c, s = st[name + "_codes"][at].int(), st[name + "_scales"][at].double()
    sign = 1.0 - 2.0 * torch.stack([c >> 3 & 1, c >> 7 & 1], -1).double()
    m = torch.stack([c & 7, c >> 4 & 7], -1).double()
    v = torch.where(m < 2, m / 2, (2 + m % 2) * torch.exp2(torch.floor(m / 2) - 2)) * sign   # 1.m 2^(e - 1), below 1 0.m
    v = v.flatten(-2) * torch.exp2(s - 127).transpose(2, 3).repeat_interleave(_BLOCK, 3)
    return v.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_read(st: dict) -> dict:
    out = {}
    for name in ("k", "v"):
        x = torch.zeros(st["b"], st["heads"], st["held"], st["d"], dtype=torch.float64, device="cuda")
        for i, n in enumerate(_held(st)):
            x[i, :, :n] = _tokens(st, name, i, n)
        out[name] = x
    return out


def _exact_attend(st: dict) -> torch.Tensor:
    q, group = st["q"].double(), st["group"]
    out = torch.empty_like(q)
    for i, (n, first) in enumerate(zip(st["lengths"].tolist(), st["starts"].tolist())):
        keys, values = _tokens(st, "k", i, n), _tokens(st, "v", i, n)
        for h in range(st["heads"]):
            kt, v = keys[h].t().contiguous(), values[h].contiguous()
            for j in range(h * group, (h + 1) * group):
                s = torch.mm(q[i, j], kt) / math.sqrt(st["d"])
                if st["causal"]:
                    s += torch.full_like(s, -math.inf).triu(first + 1)
                out[i, j] = torch.mm(torch.softmax(s, 1), v)
    return out


def exact(case: dict, seed: int):
    if case["kind"] == "attend" and case["b"] * case["heads"] * case["group"] > 4096:
        return None   # thousands of small products: over the time that this may take
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "store":
            return {"k": _nearest4(st["k"].double()), "v": _nearest4(st["v"].double())}
        return {"rotate": _exact_rotate, "read": _exact_read, "attend": _exact_attend}[case["kind"]](st)
