"""The 8-bit operators of a transformer block as programs call them: the RMS norm with the
residual's addition and an 8-bit output, the product of 8-bit operands with a scale for each
block of 128, the cache of keys and values in 8 bits with a scale for each page of 64 tokens
and head, and the attention that reads it.

8-bit values are OCP e4m3 codes times a power of two held in one byte (E8M0, ``2^(b - 127)``),
the least with which the block's largest magnitude does not pass 448.
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

_PKG = "lesiondiffusion-mlx_amd"
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
_BLOCK = 128   # columns of a row that share a scale
_PAGE = 64     # tokens of a cache page


def listed() -> list[dict]:
    return [
        # The norm in front of a projection while one token is produced at a time: the smallest call,
        # where the launch and the host path count.
        {"name": "norm_token", "kind": "norm", "dtype": "fp16", "rows": 1, "c": 512, "residual": True, "quantize": True},
        # A text encoder's or UNet level's tokens of an odd width, normalised into the network's type.
        {"name": "norm_odd", "kind": "norm", "dtype": "fp32", "rows": 1601, "c": 1000, "residual": False,
         "quantize": False},
        # Prefill of a wide block: residual stream updated, 8-bit rows for the projection that follows.
        {"name": "norm_wide", "kind": "norm", "dtype": "bf16", "rows": 16384, "c": 4096, "residual": True,
         "quantize": True},
        # A projection for four tokens of one step: the weight's bytes decide.
        {"name": "dense_tokens", "kind": "dense", "dtype": "bf16", "m": 4, "k": 4096, "o": 4096, "bias": False,
         "residual": True, "act": ""},
        # 77 text tokens of 768 features to 512: the context projection of the attention benchmark.
        {"name": "dense_text", "kind": "dense", "dtype": "fp16", "m": 77, "k": 768, "o": 512, "bias": True,
         "residual": False, "act": ""},
        # Feed-forward of a UNet level's tokens, an odd width with the GELU.
        {"name": "dense_gelu", "kind": "dense", "dtype": "fp16", "m": 1600, "k": 1000, "o": 2056, "bias": True,
         "residual": False, "act": "gelu"},
        # Prefill of a wide block's feed-forward: bound by the matrix units.
        {"name": "dense_wide", "kind": "dense", "dtype": "bf16", "m": 8192, "k": 4096, "o": 8192, "bias": False,
         "residual": False, "act": ""},
        # One new token for each of 48 sequences of unequal lengths: pages partly filled, scales that rise.
        {"name": "append_tokens", "kind": "append", "dtype": "bf16", "b": 48, "heads": 8, "d": 128, "n": 1,
         "held": 2000},
        # A prompt of an odd length written behind tokens that are held already.
        {"name": "append_prompt", "kind": "append", "dtype": "fp16", "b": 2, "heads": 8, "d": 64, "n": 4001,
         "held": 100},
        # One sequence, one query, a few pages: the smallest attention call.
        {"name": "attend_token", "kind": "attend", "dtype": "fp16", "b": 1, "heads": 8, "group": 1, "d": 64, "lq": 1,
         "held": 300, "causal": False},
        # One step of 32 sequences of unequal lengths with grouped heads: the cache's bytes decide.
        {"name": "attend_batch", "kind": "attend", "dtype": "bf16", "b": 32, "heads": 8, "group": 4, "d": 128, "lq": 1,
         "held": 8192, "causal": True},
        # A prompt's part of 2,000 queries behind held tokens, causal: bound by the matrix units.
        {"name": "attend_prompt", "kind": "attend", "dtype": "fp16", "b": 1, "heads": 4, "group": 4, "d": 64,
         "lq": 2000, "held": 8000, "causal": True},
    ]


# ------------------------------------------------------------------ drawn cases

def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo: int, hi: int) -> int:
    """A feature width: mostly a multiple of 64, now and then any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 else max(64, n // 64 * 64)


def draw(rng) -> dict:
    kind = rng.choice(["norm", "dense", "dense", "append", "attend", "attend"])
    dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
    if kind == "norm":
        c = _width(rng, 64, 8192)
        rows = _log(rng, 1, min(16384, 60_000_000 // c))
        return {"kind": kind, "dtype": dtype, "rows": rows, "c": c, "residual": rng.random() < 0.6,
                "quantize": rng.random() < 0.6}
    if kind == "dense":
        k, o = _width(rng, 64, 8192), _width(rng, 64, 8192)
        m = _log(rng, 1, min(8192, 270_000_000_000 // (k * o)))
        return {"kind": kind, "dtype": dtype, "m": m, "k": k, "o": o, "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.3, "act": rng.choice(["", "", "gelu", "silu"])}
    d = rng.choice([32, 64, 64, 128, 128, 256])
    heads = rng.choice([1, 2, 4, 8, 16])
    if kind == "append":
        b = _log(rng, 1, 64)
        n = rng.choice([1, 1, _log(rng, 2, 4096)])
        n = max(1, min(n, 16_000_000 // (b * heads * d)))
        held = _log(rng, 1, max(2, min(4096, 60_000_000 // (b * heads * d))))
        return {"kind": kind, "dtype": dtype, "b": b, "heads": heads, "d": d, "n": n, "held": held}
    dtype = rng.choice(["fp16", "bf16"])
    group = rng.choice([1, 1, 2, 4, 8])
    if rng.random() < 0.65:
        b, lq = _log(rng, 1, 64), rng.choice([1, 1, 1, rng.randint(2, 8)])
        held = _log(rng, 1, max(2, min(100_000, 260_000_000 // (b * heads * d))))
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


def _blocks(features: int) -> int:
    return -(-features // _BLOCK)


def _exponent(amax: torch.Tensor) -> torch.Tensor:
    """The scale byte of blocks whose largest magnitude is ``amax`` (fp32), as int32."""
    bits = amax.view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp(min=1)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^(e - 127) in fp32 for int32 ``e`` of 1 to 254."""
    return (e << 23).view(torch.float32)


def _rows8(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows as e4m3 codes (columns padded to whole blocks) and E8M0 scales (padded to four)."""
    rows, c = y.shape
    kb = _blocks(c)
    y = torch.nn.functional.pad(y, (0, kb * _BLOCK - c)).reshape(rows, kb, _BLOCK)
    e = _exponent(y.abs().amax(2))
    codes = (y * _pow2(254 - e)[:, :, None]).to(torch.float8_e4m3fn).reshape(rows, kb * _BLOCK)
    e = torch.nn.functional.pad(e, (0, -kb % 4), value=127)
    return codes, e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _wide(codes: torch.Tensor, scales: torch.Tensor, features: int, dtype: torch.dtype) -> torch.Tensor:
    """The values that rows of codes and scales stand for."""
    rows, kb = codes.shape[0], _blocks(features)
    s = _pow2(scales.view(torch.uint8)[:, :kb].to(torch.int32)).to(dtype)
    return (codes.to(dtype).reshape(rows, kb, _BLOCK) * s[:, :, None]).reshape(rows, -1)[:, :features]


def _activations(rows: int, c: int, g: torch.Generator) -> torch.Tensor:
    """~N(0, 1) with a few loud columns, as residual streams have them."""
    x = torch.randn(rows, c, generator=g, device="cuda")
    x[:, :: 97] *= 8.0
    return x


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    t = _DTYPES[case["dtype"]]
    st = dict(case)
    if case["kind"] == "norm":
        st["x"] = _activations(case["rows"], case["c"], g).to(t)
        st["r"] = _activations(case["rows"], case["c"], g).to(t) if case["residual"] else None
        st["gamma"] = 1 + 0.1 * torch.randn(case["c"], generator=g, device="cuda")
        return st
    if case["kind"] == "dense":
        m, k, o = case["m"], case["k"], case["o"]
        st["codes"], st["scales"] = _rows8(_activations(m, k, g))
        st["w_codes"], st["w_scales"] = _rows8(torch.randn(o, k, generator=g, device="cuda") / math.sqrt(k))
        st["b"] = 0.1 * torch.randn(o, generator=g, device="cuda") if case["bias"] else None
        st["r"] = torch.randn(m, o, generator=g, device="cuda").to(t) if case["residual"] else None
        return st
    b, h, d, held = case["b"], case["heads"], case["d"], _held(case)
    new = case["n"] if case["kind"] == "append" else case["lq"]
    width = -(-(max(held) + new) // _PAGE)
    pages = b * width + 1   # the last page is in no table
    loud = 1 + 3 * torch.rand(h, 1, d, generator=g, device="cuda")
    k = torch.randn(pages, h, _PAGE, d, generator=g, device="cuda") * loud
    v = torch.randn(pages, h, d, _PAGE, generator=g, device="cuda")
    for name, c in (("k", k), ("v", v)):
        e = _exponent(c.abs().amax((2, 3)))
        st[name + "_codes"] = (c * _pow2(254 - e)[:, :, None, None]).to(torch.float8_e4m3fn)
        st[name + "_scales"] = e.to(torch.uint8).view(torch.float8_e8m0fnu)
    del k, v, c
    st["table"] = torch.randperm(pages - 1, generator=g, device="cuda").to(torch.int32).reshape(b, width)
    st["starts"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    st["lengths"] = st["starts"] + new
    if case["kind"] == "append":
        st["k"] = (torch.randn(b, h, new, d, generator=g, device="cuda") * 1.5 * loud).to(t)
        st["v"] = (torch.randn(b, h, new, d, generator=g, device="cuda") * 1.5).to(t)
    else:
        st["q"] = torch.randn(b, h * case["group"], new, d, generator=g, device="cuda").to(t)
    return st


# ------------------------------------------------------------------ plain forms

def _norm(st: dict) -> dict:
    out = {}
    x = st["x"]
    if st["r"] is not None:
        x = out["sum"] = (x.float() + st["r"].float()).to(x.dtype)
    f = x.float()
    y = f * torch.rsqrt((f * f).mean(1, keepdim=True) + 1e-6) * st["gamma"]
    if st["quantize"]:
        out["codes"], out["scales"] = _rows8(y)
    else:
        out["y"] = y.to(x.dtype)
    return out


def _activation(y: torch.Tensor, act: str) -> torch.Tensor:
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y * torch.sigmoid(y) if act == "silu" else y


def _dense(st: dict) -> torch.Tensor:
    a = _wide(st["codes"], st["scales"], st["k"], torch.float32)
    w = _wide(st["w_codes"], st["w_scales"], st["k"], torch.float32)
    y = a @ w.t()
    if st["b"] is not None:
        y = y + st["b"]
    if st["r"] is not None:
        y = y + st["r"].float()
    return _activation(y, st["act"]).to(_DTYPES[st["dtype"]])


def _put(codes: torch.Tensor, scales: torch.Tensor, new: torch.Tensor, st: dict, turned: bool) -> None:
    """Write ``new`` (B, H, n, D) at ``starts`` into pages of (64, D) codes, or (D, 64) where ``turned``."""
    b, h, n, d = new.shape
    starts, table = st["starts"].long(), st["table"].long()
    nb = (n + 2 * _PAGE - 2) // _PAGE
    slot = starts[:, None] // _PAGE + torch.arange(nb, device=new.device)
    pos = slot[:, :, None] * _PAGE + torch.arange(_PAGE, device=new.device)            # (B, nb, 64)
    src = pos - starts[:, None, None]
    touched = slot * _PAGE < (starts + n)[:, None]
    page = torch.where(touched, table.gather(1, slot.clamp(max=table.shape[1] - 1)), codes.shape[0] - 1)
    rows = torch.arange(b, device=new.device)[:, None]
    tok = new.transpose(1, 2)[rows, src.clamp(0, n - 1).reshape(b, -1)].float()
    tok = tok.reshape(b, nb, _PAGE, h, d).transpose(2, 3)                              # (B, nb, H, 64, D)
    raw, byte = codes.view(torch.uint8)[page], scales.view(torch.uint8)[page].to(torch.int32)
    held = raw.transpose(3, 4) if turned else raw                                      # (B, nb, H, 64, D)
    is_new = ((src >= 0) & (src < n))[:, :, None, :, None]
    need = _exponent(torch.where(is_new, tok.abs(), 0.0).amax((3, 4)))
    has_old = (slot * _PAGE < starts[:, None])[:, :, None]
    to = torch.where(has_old, torch.maximum(need, byte), need)
    was = held.contiguous().view(torch.float8_e4m3fn).float() * _pow2(byte)[..., None, None]
    val = torch.where(is_new, tok, was) * _pow2(254 - to)[..., None, None]
    keep = (src >= n)[:, :, None, :, None] | ~touched[:, :, None, None, None]
    fresh = torch.where(keep, held, val.to(torch.float8_e4m3fn).view(torch.uint8))
    codes.view(torch.uint8)[page] = fresh.transpose(3, 4) if turned else fresh
    scales.view(torch.uint8)[page] = torch.where(touched[:, :, None], to, byte).to(torch.uint8)


def _append(st: dict) -> dict:
    _put(st["k_codes"], st["k_scales"], st["k"], st, False)
    _put(st["v_codes"], st["v_scales"], st["v"], st, True)
    return {n: st[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales")}


def _attend(st: dict) -> torch.Tensor:
    q, table, scale = st["q"], st["table"].long(), st["d"] ** -0.5
    b, hq, lq, d = q.shape
    h, n = st["heads"], table.shape[1] * _PAGE
    ks = _pow2(st["k_scales"].view(torch.uint8)[table].to(torch.int32))[..., None, None]   # (B, W, H, 1, 1)
    vs = _pow2(st["v_scales"].view(torch.uint8)[table].to(torch.int32))[..., None, None]
    k = st["k_codes"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * ks       # (B, W, H, 64, D)
    v = st["v_codes"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * vs       # (B, W, H, D, 64)
    k = k.permute(0, 2, 4, 1, 3).reshape(b, h, d, n)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, h, n, d)
    s = torch.matmul(q.float().reshape(b, h, hq // h * lq, d), k).reshape(b, h, hq // h, lq, n) * scale
    key = torch.arange(n, device=q.device)
    seen = key < st["lengths"][:, None, None]
    if st["causal"]:
        seen = seen & (key <= st["starts"][:, None, None] + torch.arange(lq, device=q.device)[:, None])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(4, keepdim=True))
    o = torch.matmul(p.reshape(b, h, hq // h * lq, n), v).reshape(b, h, hq // h, lq, d) / p.sum(4, keepdim=True)
    return o.reshape(b, hq, lq, d).to(q.dtype)


def run(st: dict):
    kind = st["kind"]
    if not own:
        return {"norm": _norm, "dense": _dense, "append": _append, "attend": _attend}[kind](st)
    ops = importlib.import_module(_PKG).ops
    if kind == "norm":
        y = ops.rms_norm(st["x"], st["gamma"], 1e-6, residual=st["r"], quantize=st["quantize"])
        out = {}
        if st["r"] is not None:
            y, out["sum"] = y
        if st["quantize"]:
            return {**out, "codes": y.codes, "scales": y.scales}
        return {**out, "y": y}
    if kind == "dense":
        return ops.dense8(ops.Quantized8(st["codes"], st["scales"], st["k"]),
                          ops.Quantized8(st["w_codes"], st["w_scales"], st["k"]), st["b"], residual=st["r"],
                          act=st["act"] or None, dtype=_DTYPES[st["dtype"]])
    cache = ops.Cache8(st["k_codes"], st["v_codes"], st["k_scales"], st["v_scales"])
    if kind == "append":
        ops.cache8_append(cache, st["k"], st["v"], st["table"], st["starts"])
        return {n: st[n] for n in ("k_codes", "k_scales", "v_codes", "v_scales")}
    return ops.cache8_attention(st["q"], cache, st["table"], st["lengths"], st["d"] ** -0.5,
                                starts=st["starts"] if st["causal"] else None)


# ------------------------------------------------------------------ the work itself

def _visible(case: dict) -> int:
    """(query, key) pairs of one head, over all sequences."""
    lq, total = case["lq"], 0
    for n in _held(case):
        total += lq * n + (lq * (lq + 1) // 2 if case["causal"] else lq * lq)
    return total


def work(case: dict) -> dict:
    size = _BYTES[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["c"]
        each = size * (3 if case["residual"] else 1) + (1 if case["quantize"] else size)
        return {"bytes": n * each + case["c"] * 4, "flops": 5 * n}
    if case["kind"] == "dense":
        m, k, o = case["m"], case["k"], case["o"]
        return {"bytes": (m + o) * (k + _blocks(k)) + m * o * size * (2 if case["residual"] else 1),
                "flops": 2 * m * k * o}
    b, h, d = case["b"], case["heads"], case["d"]
    if case["kind"] == "append":
        n = b * h * case["n"] * d
        return {"bytes": 2 * n * (size + 1), "flops": 4 * n}
    keys = sum(_held(case)) + b * case["lq"]
    rows = b * h * case["group"] * case["lq"]
    return {"bytes": 2 * keys * h * d + 2 * rows * d * size,
            "flops": 4 * h * case["group"] * d * _visible(case)}


# ------------------------------------------------------------------ 64-bit results

def _exact_scale(amax: torch.Tensor) -> torch.Tensor:
    """The least power of two from 2^-126 on with amax <= 448 * it, in float64."""
    e = torch.ceil(torch.log2(torch.clamp(amax, min=1e-300) / 448.0)).clamp(min=-126)
    e = torch.where(448.0 * torch.exp2(e - 1) >= amax, e - 1, e).clamp(min=-126)
    return torch.where(448.0 * torch.exp2(e) < amax, e + 1, e)


def _nearest8(v: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each ``v`` (|v| <= 448), ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_norm(st: dict) -> dict:
    out = {}
    x = st["x"]
    if st["r"] is not None:
        total = x.double() + st["r"].double()
        out["sum"] = total
        x = total.to(x.dtype)   # what the norm reads is the stored sum
    x = x.double()
    y = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / x.shape[1] + 1e-6) * st["gamma"].double()
    if not st["quantize"]:
        return {**out, "y": y}
    kb = _blocks(y.shape[1])
    full = torch.zeros(y.shape[0], kb * _BLOCK, dtype=torch.float64, device=y.device)
    full[:, :y.shape[1]] = y
    full = full.reshape(-1, kb, _BLOCK)
    e = _exact_scale(full.abs().max(2).values)
    scales = torch.ones(y.shape[0], -(-kb // 4) * 4, dtype=torch.float64, device=y.device)
    scales[:, :kb] = torch.exp2(e)
    return {**out, "codes": _nearest8(full / torch.exp2(e)[:, :, None]).reshape(y.shape[0], -1), "scales": scales}


def _exact_dense(st: dict) -> torch.Tensor:
    a = st["codes"].double()
    w = st["w_codes"].double()
    for c, s in ((a, st["scales"]), (w, st["w_scales"])):
        for j in range(_blocks(st["k"])):
            c[:, j * _BLOCK:(j + 1) * _BLOCK] *= s[:, j:j + 1].double()
    y = torch.mm(a, w.t().contiguous())
    if st["b"] is not None:
        y += st["b"].double()
    if st["r"] is not None:
        y += st["r"].double()
    if st["act"] == "gelu":
        return y * torch.special.ndtr(y)
    return y / (1 + torch.exp(-y)) if st["act"] == "silu" else y


def _exact_append(st: dict) -> dict:
    out = {}
    table, starts = st["table"].tolist(), st["starts"].tolist()
    for name, turned in (("k", False), ("v", True)):
        codes, scales = st[name + "_codes"].double(), st[name + "_scales"].double()
        if turned:
            codes = codes.transpose(2, 3).contiguous()
        new = st[name].double()
        for i, first in enumerate(starts):
            last = first + st["n"]
            for slot in range(first // _PAGE, -(-last // _PAGE)):
                page, lo, hi = table[i][slot], max(first - slot * _PAGE, 0), min(last - slot * _PAGE, _PAGE)
                put = new[i][:, slot * _PAGE + lo - first: slot * _PAGE + hi - first]       # (H, tokens, D)
                to = torch.exp2(_exact_scale(put.abs().amax((1, 2))))
                if lo:
                    to = torch.maximum(to, scales[page])
                    codes[page][:, :lo] = _nearest8(codes[page][:, :lo] * (scales[page] / to)[:, None, None])
                codes[page][:, lo:hi] = _nearest8(put / to[:, None, None])
                scales[page] = to
        out[name + "_codes"], out[name + "_scales"] = codes.transpose(2, 3) if turned else codes, scales
    return out


def _exact_attend(st: dict) -> torch.Tensor:
    q, group = st["q"].double(), st["group"]
    out = torch.empty_like(q)
    for i, (n, first) in enumerate(zip(st["lengths"].tolist(), st["starts"].tolist())):
        at = st["table"][i, :-(-n // _PAGE)].long()
        for h in range(st["heads"]):
            k = st["k_codes"][at, h].double() * st["k_scales"][at, h].double()[:, None, None]
            v = st["v_codes"][at, h].double() * st["v_scales"][at, h].double()[:, None, None]
            k, v = k.reshape(-1, st["d"])[:n], v.transpose(1, 2).reshape(-1, st["d"])[:n]
            kt = k.t().contiguous()
            for j in range(h * group, (h + 1) * group):
                s = torch.mm(q[i, j], kt) / math.sqrt(st["d"])
                if st["causal"]:
                    s += torch.full_like(s, -math.inf).triu(first + 1)
                out[i, j] = torch.mm(torch.softmax(s, 1), v)
    return out


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "attend" and case["b"] * case["heads"] * case["group"] > 4096:
        return None   # thousands of small products: over the time that this may take
    with torch.no_grad():
        return {"norm": _exact_norm, "dense": _exact_dense, "append": _exact_append, "attend": _exact_attend}[
            case["kind"]](st)
