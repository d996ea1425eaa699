"""The 8-bit operators: RMS norm with residual and 8-bit rows, the block-scaled e4m3 product, the paged
8-bit cache and its attention. Refusals through the C ABI run on the CPU; results are compared with
float64 on an MI355X."""

from __future__ import annotations

import ctypes
import math
import subprocess

import pytest
import torch

from tests.conftest import REPO

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
NAN = math.nan


# ------------------------------------------------------------------ float64 reference

def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def tiny(t: torch.dtype) -> float:
    """Half the spacing of ``t``'s subnormal numbers."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def scale_for(amax: torch.Tensor) -> torch.Tensor:
    """The least 2^e, e >= -126, with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax)                      # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), 2.0 ** -126)


def nearest8(v: torch.Tensor) -> torch.Tensor:
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def rows8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of float64 rows, blocks of 128 padded with zeros."""
    c = x.shape[-1]
    kb = -(-c // 128)
    x = torch.nn.functional.pad(x.double(), (0, kb * 128 - c)).unflatten(-1, (kb, 128))
    s = scale_for(x.abs().amax(-1))
    return nearest8(x / s[..., None]).flatten(-2), s


def wide(q) -> torch.Tensor:
    kb = q.codes.shape[-1] // 128
    v = q.codes.cpu().double().unflatten(-1, (kb, 128)) * q.scales.cpu().double()[..., :kb, None]
    return v.flatten(-2)[..., :q.features]


def rand(shape, seed, t=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(t)


# ------------------------------------------------------------------ refusals on the CPU

def test_structs_match_c_layout(pkg, tmp_path) -> None:
    lib = pkg._lib
    fields = {"ldx_rms_norm_args": lib.RmsNormArgs, "ldx_dense8_args": lib.Dense8Args, "ldx_cache8": lib.Cache8Block,
              "ldx_cache8_append_args": lib.Cache8AppendArgs, "ldx_cache8_attention_args": lib.Cache8AttentionArgs}
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "ldx.h"', "int main(void) {"]
    for cname, cls in fields.items():
        src.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        src += [f'printf("{cname} {f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in cls._fields_]
    src.append(f'printf("consts block8 %d\\nconsts page8 %d\\n", LDX_BLOCK8, LDX_PAGE8); return 0; }}')
    (tmp_path / "l.c").write_text("\n".join(src))
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        cname, what, val = line.split()
        if cname == "consts":
            want = {"block8": lib.BLOCK8, "page8": lib.PAGE8}[what]
        else:
            want = ctypes.sizeof(fields[cname]) if what == "size" else getattr(fields[cname], what).offset
        assert int(val) == want, line


def refused(pkg, rc: int, word: str) -> None:
    assert rc == pkg._lib.LDX_EINVAL
    assert word in pkg._lib.last_error(), pkg._lib.last_error()


@pytest.mark.parametrize("bad", [
    {"x": None}, {"gamma": None}, {"y": None}, {"rows": 0}, {"features": 0}, {"dtype": 3}, {"x_pitch": 99},
    {"y_pitch": 99}, {"eps": 0.0}, {"eps": NAN}, {"codes": 16}, {"sum": 16, "sum_pitch": 100},
    {"residual": 16, "residual_pitch": 9}, {"residual": 16, "residual_pitch": 100, "sum": 16, "sum_pitch": 9},
    {"y": None, "codes": 16, "codes_pitch": 112, "scales": 16, "scales_pitch": 4},
    {"y": None, "codes": 16, "codes_pitch": 128, "scales": 16, "scales_pitch": 2},
    {"y": None, "codes": 8, "codes_pitch": 128, "scales": 16, "scales_pitch": 4},
    {"y": None, "codes": 16, "codes_pitch": 128, "scales": None, "scales_pitch": 4},
])
def test_rms_norm_refuses(pkg, bad) -> None:
    a = pkg._lib.RmsNormArgs(rows=2, features=100, dtype=0, x=16, x_pitch=100, gamma=16, eps=1e-6, y=16, y_pitch=100)
    for k, v in bad.items():
        setattr(a, k, v)
    refused(pkg, pkg._lib.lib.ldx_rms_norm(ctypes.byref(a), None), "rms_norm")


def test_quantize8_refuses(pkg) -> None:
    q = pkg._lib.lib.ldx_quantize8
    for args in ((None, 8, 1, 8, 0, 16, 128, 16, 4), (16, 7, 1, 8, 0, 16, 128, 16, 4), (16, 8, 0, 8, 0, 16, 128, 16, 4),
                 (16, 8, 1, 8, 5, 16, 128, 16, 4), (16, 8, 1, 8, 0, 16, 64, 16, 4), (16, 8, 1, 8, 0, 16, 128, 16, 1),
                 (16, 8, 1, 8, 0, 16, 128, 18, 4)):
        refused(pkg, q(*args, None), "quantize8")


@pytest.mark.parametrize("bad", [
    {"rows": 0}, {"features": 0}, {"out_features": 0}, {"dtype": 4}, {"act": 3}, {"x_codes": None}, {"w_scales": None},
    {"y": None}, {"x_pitch": 128}, {"w_pitch": 264}, {"x_scales_pitch": 3}, {"w_codes": 24}, {"x_scales": 2},
    {"y_pitch": 4}, {"residual": 16, "residual_pitch": 4}, {"rows": 0x7fffffff, "out_features": 1 << 20, "y_pitch": 1 << 20},
    {"rows": 0x7fffffff, "out_features": 300, "y_pitch": 300},
    {"features": 1 << 22 | 1, "x_pitch": 1 << 23, "w_pitch": 1 << 23, "x_scales_pitch": 1 << 20, "w_scales_pitch": 1 << 20},
    {"w_pitch": (1 << 22) + 16}, {"w_scales_pitch": (1 << 22) + 4},
])
def test_dense8_refuses(pkg, bad) -> None:
    a = pkg._lib.Dense8Args(rows=3, features=200, out_features=5, x_codes=16, x_pitch=256, x_scales=16, x_scales_pitch=4,
                            w_codes=16, w_pitch=256, w_scales=16, w_scales_pitch=4, y=16, y_pitch=5)
    for k, v in bad.items():
        setattr(a, k, v)
    refused(pkg, pkg._lib.lib.ldx_dense8(ctypes.byref(a), None), "dense8")


def _cache_args(lib, **kw):
    c = dict(k=16, v=16, k_scales=1, v_scales=1, pages=2, heads=2, head_dim=64)
    c.update({k: v for k, v in kw.items() if k in c})
    return lib.Cache8Block(**c)


@pytest.mark.parametrize("bad", [
    {"pages": 0}, {"heads": 0}, {"head_dim": 48}, {"head_dim": 512}, {"k_scales": None}, {"tokens": 0}, {"tokens": (1 << 28) + 1}, {"batch": 0},
    {"batch": 70000}, {"width": 0}, {"table_pitch": 0}, {"table": None}, {"starts": None}, {"dtype": 9}, {"src": None},
])
def test_cache8_append_refuses(pkg, bad) -> None:
    lib = pkg._lib
    a = lib.Cache8AppendArgs(cache=_cache_args(lib, **bad), batch=1, tokens=1, k=16, v=16, table=16, table_pitch=1,
                             width=1, starts=16)
    for k, v in bad.items():
        if k == "src":
            a.v = v
        elif hasattr(a, k):
            setattr(a, k, v)
    refused(pkg, lib.lib.ldx_cache8_append(ctypes.byref(a), None), "cache8_append")


@pytest.mark.parametrize("bad", [
    {"pages": 0}, {"head_dim": 16}, {"q_heads": 3}, {"q_heads": 0}, {"q_len": 0}, {"batch": 0}, {"width": 0},
    {"width": 1 << 25, "table_pitch": 1 << 25}, {"table_pitch": 0}, {"lengths": None}, {"dtype": 1}, {"scale": NAN},
    {"src": None}, {"q_len": 1 << 30}, {"q_len": 1 << 27},
])
def test_cache8_attention_refuses(pkg, bad) -> None:
    lib = pkg._lib
    a = lib.Cache8AttentionArgs(cache=_cache_args(lib, **bad), batch=1, q_heads=2, q_len=1, q=16, o=16, scale=1.0,
                                table=16, table_pitch=1, width=1, lengths=16)
    for k, v in bad.items():
        if k == "src":
            a.q = v
        elif hasattr(a, k):
            setattr(a, k, v)
    assert lib.lib.ldx_cache8_attention_workspace_bytes(ctypes.byref(a)) == 0
    refused(pkg, lib.lib.ldx_cache8_attention(ctypes.byref(a), None), "cache8_attention")


def test_attention_workspace_is_bounded(pkg) -> None:
    """Partial results are at most 256 MiB, whatever a call's size, and nothing where the queries fill the card many
    times over; long sequences of few queries are still spread over workgroups."""
    lib = pkg._lib

    def parts(batch, heads, group, q_len, d, width):
        a = lib.Cache8AttentionArgs(cache=_cache_args(lib, heads=heads, head_dim=d), batch=batch, q_heads=heads * group,
                                    q_len=q_len, q=16, o=16, scale=1.0, table=16, table_pitch=width, width=width, lengths=16)
        n = lib.lib.ldx_cache8_attention_workspace_bytes(ctypes.byref(a))
        per = batch * heads * group * q_len * (d + 2) * 4
        assert n % per == 0 and n <= 256 << 20, (batch, heads, group, q_len, d, width, n)
        return max(n // per, 1)

    assert parts(16, 8, 4, 4000, 64, 126) == parts(64, 8, 4, 4096, 64, 64) == parts(16, 8, 8, 15900, 256, 440) == 1
    assert parts(1, 4, 4, 2000, 64, 157) > 1 and parts(1, 8, 1, 1, 128, 128) > 1 and parts(1, 1, 1, 128, 64, 20000) > 1
    gen = torch.Generator().manual_seed(1)
    log = lambda lo, hi: int(math.exp(math.log(lo) + torch.rand((), generator=gen).item() * math.log(hi / lo)))
    for _ in range(3000):
        d = [32, 64, 128, 256][log(1, 16) % 4]
        batch, heads, group = log(1, 2000), log(1, 64), log(1, 16)
        parts(batch, heads, group, max(1, min(log(1, 100_000), 0x7fffffff // (batch * heads * group))), d, log(1, 1 << 24))


def test_cpu_tensors_are_refused(pkg) -> None:
    ops = pkg.ops
    x = torch.zeros(2, 8)
    q = ops.Quantized8.empty((2,), 8, x)
    cache = ops.Cache8.empty(2, 1, 32, device="cpu")
    ints = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.quantize8(x), lambda: ops.rms_norm(x, torch.ones(8)), lambda: ops.dense8(q, q),
                 lambda: ops.cache8_append(cache, x, x, ints, ints),
                 lambda: ops.cache8_attention(x, cache, ints, ints, 1.0)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="Quantized8"):
        ops.dense8(x, q)
    with pytest.raises(ValueError, match="Cache8"):
        ops.cache8_attention(x, x, ints, ints, 1.0)


def test_sizes_beyond_the_abi_fields_are_refused(pkg, monkeypatch) -> None:
    """Features, tokens, batches and table widths that the C structs' 32 bits do not hold, none of which a call may
    take for the rest of them; tensors without memory stand in for those of a device."""
    ops = pkg.ops
    monkeypatch.setattr(ops, "_need", lambda *a: None)
    meta = lambda *shape, t=torch.float16: torch.empty(shape, dtype=t, device="meta")
    huge = (1 << 32) + 8
    ints32 = lambda *shape: meta(*shape, t=torch.int32)
    codes, scales = meta(2, 1, 64, 32, t=torch.float8_e4m3fn), meta(2, 1, t=torch.float8_e8m0fnu)
    cache = ops.Cache8(codes, codes.view(2, 1, 32, 64), scales, scales)
    monkeypatch.setattr(ops, "_cache_block", lambda c, what: (pkg._lib.Cache8Block(16, 16, 1, 1, 2, 1, 32), 0))
    kv = meta(1, 1, 1, 32).expand(1, 1, huge, 32)
    many = meta(1, 1, 1, 32).expand(huge, 1, 1, 32)
    one = meta(1, 1, 1, 32)
    for word, call in (
            ("features", lambda: ops.quantize8(meta(1, huge))), ("features", lambda: ops.rms_norm(meta(1, huge), meta(huge))),
            ("tokens", lambda: ops.cache8_append(cache, kv, kv, ints32(1, 1), ints32(1))),
            ("tokens", lambda: ops.cache8_append(cache, many, many, ints32(huge, 1), ints32(huge))),
            ("pages", lambda: ops.cache8_append(cache, one, one, ints32(1, huge), ints32(1))),
            ("pages", lambda: ops.cache8_attention(one, cache, ints32(1, huge), ints32(1), 1.0)),
            ("queries", lambda: ops.cache8_attention(kv, cache, ints32(1, 1), ints32(1), 1.0, out=kv)),
            ("queries", lambda: ops.cache8_attention(many, cache, ints32(huge, 1), ints32(huge), 1.0, out=many))):
        with pytest.raises(ValueError, match=word):
            call()


# ------------------------------------------------------------------ 8-bit rows and the norm

SHAPES = [(1, 1), (3, 7), (1, 128), (2, 129), (5, 512), (4, 513), (7, 1000), (3, 1024), (2, 2047), (2, 4096), (1, 5001),
          (2, 8200), (1, 20011)]


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize8_is_the_nearest_code(pkg, dev, shape, t) -> None:
    """Scaling by a power of two is exact, so codes and scales equal the float64 ones."""
    x = rand(shape, sum(shape), t) * torch.exp2(torch.randint(-6, 6, shape, generator=torch.Generator().manual_seed(1)).float()).to(t)
    x[..., -1:] = 0
    q = pkg.ops.quantize8(x.to(dev))
    codes, s = rows8(x)
    kb = s.shape[-1]
    assert q.codes.shape == codes.shape and q.scales.shape[-1] == -(-kb // 4) * 4
    assert torch.equal(q.codes.cpu().double(), codes)
    assert torch.equal(q.scales.cpu().double()[..., :kb], s)
    assert (q.scales.cpu().double()[..., kb:] == 1).all()
    assert torch.equal(q.float().cpu().double(), wide(q))


@gpu
def test_quantize8_of_special_values(pkg, dev) -> None:
    """All-zero blocks, the ends of fp32, ties, 448's neighbours; NaN stays NaN beside numbers that keep
    their scale, an infinity becomes NaN."""
    x = torch.zeros(8, 128)
    x[1] = torch.linspace(-448, 448, 128)
    x[2, 0], x[2, 1] = 449.0, -1.0
    x[3, :2] = torch.tensor([3.0e38, -1.0e30])
    x[4, :3] = torch.tensor([2.0 ** -140, -2.0 ** -126, 2.0 ** -130])
    x[5] = torch.arange(128) * 0.0625 + 16.0          # ties among them
    x[6, :3] = torch.tensor([NAN, 448.0, -3.0])
    x[7, :2] = torch.tensor([math.inf, 5.0])
    q = pkg.ops.quantize8(x.to(dev))
    got, s = q.codes.cpu().double(), q.scales.cpu().double()[:, 0]
    codes, want = rows8(x[:6])
    assert torch.equal(got[:6], codes) and torch.equal(s[:6], want[:, 0])
    assert got[6, 0].isnan() and got[6, 1] == 448 and got[6, 2] == -3 and s[6] == 1
    assert got[7, 0].isnan() and got[7, 1] == 0 and (got[7, 2:] == 0).all()


def norm_reference(x, gamma, eps, r):
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    d = s.double()
    return s, d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * gamma.double()


def norm_relative(c: int) -> float:
    """Roundings of the norm in fp32, relative: the squares' sum takes at most c / 256 + 80 in a row (a
    thread's own, then six levels of lanes and four waves) and half of its error reaches the root; the
    mean, eps, root, quotient and two products take one each."""
    return ((c / 256 + 80) / 2 + 6) * 2.0 ** -24


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm_matches_float64(pkg, dev, shape, residual, t) -> None:
    c = shape[-1]
    x, gamma = rand(shape, 3 + c, t, 2.0), 1 + rand((c,), 4, scale=0.1)
    r = rand(shape, 5, t) if residual else None
    s, y = norm_reference(x, gamma, 1e-6, r)
    rd = None if r is None else r.to(dev)
    got = pkg.ops.rms_norm(x.to(dev), gamma.to(dev), 1e-6, residual=rd)
    if residual:
        got, total = got
        assert torch.equal(total.cpu(), s)
    err = (got.cpu().double() - y).abs()
    rel = norm_relative(c)
    assert (err <= y.abs() * (half_step(t) * (1 + rel) + rel) + tiny(t)).all(), (err / y.abs()).max()
    q = pkg.ops.rms_norm(x.to(dev), gamma.to(dev), 1e-6, residual=rd, quantize=True)
    if residual:
        q, total = q
        assert torch.equal(total.cpu(), s)
    # Scales: least for an amax that is off by `rel`; codes: within half a step of the value they round.
    kb = -(-c // 128)
    blocks = torch.nn.functional.pad(y, (0, kb * 128 - c)).unflatten(-1, (kb, 128))
    amax, sc = blocks.abs().amax(-1), q.scales.cpu().double()[..., :kb]
    assert ((448 * sc >= amax * (1 - rel)) & ((448 * sc / 2 < amax * (1 + rel)) | (sc == 2.0 ** -126))).all()
    v = blocks / sc[..., None]
    code = q.codes.cpu().double().unflatten(-1, (kb, 128))
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6) * (1 + rel))) - 3)
    assert ((code - v).abs() <= step / 2 + v.abs() * rel).all()


@gpu
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [3.0e19, 2.0 ** 127])
@pytest.mark.parametrize("c", [100, 3000, 9000])
def test_rms_norm_of_values_whose_squares_overflow(pkg, dev, c, size, t) -> None:
    x = (rand((3, c), c) / 8).clamp(-1, 1)
    x[:, 0] = 1.0
    x = (x * size).to(t)
    x[1] = rand((c,), 1).to(t)
    _, y = norm_reference(x, torch.ones(c), 1e-6, None)
    got = pkg.ops.rms_norm(x.to(dev), torch.ones(c, device=dev), 1e-6).cpu().double()
    rel = norm_relative(c)
    assert ((got - y).abs() <= y.abs() * (half_step(t) * (1 + rel) + rel) + tiny(t)).all()


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("c", [8193, 65536, (1 << 20) + 3, (1 << 24) + 1])
def test_rms_norm_of_long_rows(pkg, dev, c, t) -> None:
    """A row's error does not grow with its length: eight squares at a time are summed in fp32 (at most eight
    roundings, half of which reach the root), the eights in fp64; root, quotient and products take four more."""
    rel = (8 / 2 + 4) * 2.0 ** -24
    gamma = (1 + rand((c,), 4, scale=0.1)).to(dev)
    x = torch.stack((torch.full((c,), 1.1), rand((c,), 5), rand((c,), 6) ** 3))
    if t != torch.float16:
        x[2] *= 1e19      # squares and their sum leave fp32
    x = x.to(t).to(dev)
    d = x.double()
    y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-6) * gamma.double()
    err = (pkg.ops.rms_norm(x, gamma).double() - y).abs()
    bar = y.abs() * (half_step(t) * (1 + rel) + rel) + tiny(t)
    assert (err <= bar).all(), (err / bar).amax(1)
    r = rand((3, c), 7, t).to(dev)
    got, s = pkg.ops.rms_norm(x, gamma, residual=r)
    assert torch.equal(s, (x.float() + r.float()).to(t)) and torch.equal(got, pkg.ops.rms_norm(s, gamma))


@gpu
def test_quantize8_of_many_rows(pkg, dev) -> None:
    """More rows than one axis of a launch takes."""
    n = (1 << 26) + 1001
    x = torch.randn(n, 3, device=dev).half()
    q = pkg.ops.quantize8(x)
    for lo in (0, (1 << 24) - 8, (1 << 26) - 500, n - 700):
        part = pkg.ops.quantize8(x[lo:lo + 700])
        m = part.codes.shape[0]
        assert torch.equal(part.codes.view(torch.uint8), q.codes[lo:lo + m].view(torch.uint8))
        assert torch.equal(part.scales.view(torch.uint8), q.scales[lo:lo + m].view(torch.uint8))


@gpu
def test_rms_norm_keeps_nan_to_its_row(pkg, dev) -> None:
    x = rand((4, 300), 1)
    x[1, 5], x[2, 7] = NAN, math.inf
    gamma = torch.ones(300, device=dev)
    clean = pkg.ops.rms_norm(x[[0, 3]].to(dev), gamma).cpu()
    y = pkg.ops.rms_norm(x.to(dev), gamma).cpu()
    assert torch.equal(y[[0, 3]], clean)
    assert y[1].isnan().all()
    assert y[2, 7].isnan() and (y[2, :7] == 0).all()     # finite / infinite norm
    q = pkg.ops.rms_norm(x.to(dev), gamma, quantize=True)
    assert q.float()[1].isnan().all() and q.float()[[0, 3]].isfinite().all()


@gpu
@pytest.mark.parametrize("c", [96, 5000, 20000])
def test_rms_norm_strides_and_in_place(pkg, dev, c) -> None:
    """Column ranges of wider tensors, odd offsets, 3-D leads; out over x, the sum over either operand."""
    t = torch.float16
    gamma = (1 + rand((c,), 2, scale=0.1)).to(dev)
    base = rand((2, 3, c + 11), 1, t).to(dev)
    x, r = base[..., 3:3 + c], rand((2, 3, c), 3, t).to(dev)
    want, total = pkg.ops.rms_norm(x.contiguous(), gamma, residual=r)
    got, s = pkg.ops.rms_norm(x, gamma, residual=r)
    assert torch.equal(got, want) and torch.equal(s, total) and s.shape == x.shape
    before = base.clone()
    got, s = pkg.ops.rms_norm(x, gamma, residual=r, sum_out=x)
    assert s is x and torch.equal(x, total) and torch.equal(got, want)
    assert torch.equal(base[..., :3], before[..., :3]) and torch.equal(base[..., 3 + c:], before[..., 3 + c:])
    y = r.clone()
    got, s = pkg.ops.rms_norm(before[..., 3:3 + c], gamma, residual=y, sum_out=y)
    assert torch.equal(y, total) and torch.equal(got, want)
    z = total.clone()
    assert pkg.ops.rms_norm(z, gamma, out=z) is z and torch.equal(z, want)
    e = pkg.ops.rms_norm(r[:, :1].expand(2, 3, c), gamma)       # broadcast rows
    assert torch.equal(e[:, 0], e[:, 2])
    q = pkg.ops.quantize8(x.transpose(0, 1))
    assert torch.equal(q.codes.view(torch.uint8), pkg.ops.quantize8(x.transpose(0, 1).contiguous()).codes.view(torch.uint8))


@gpu
def test_norm_refuses_on_the_device(pkg, dev) -> None:
    ops = pkg.ops
    x, g = torch.zeros(2, 8, device=dev), torch.ones(8, device=dev)
    for call in (lambda: ops.rms_norm(x, g[:4]), lambda: ops.rms_norm(x, g, residual=x.half()),
                 lambda: ops.rms_norm(x, g, residual=x[:1]), lambda: ops.rms_norm(x, g, out=x[:, :4]),
                 lambda: ops.rms_norm(x, g, out=x.clone(), quantize=True), lambda: ops.rms_norm(x, g, sum_out=x),
                 lambda: ops.rms_norm(x, g, eps=0.0), lambda: ops.rms_norm(x.long(), g), lambda: ops.quantize8(x[:0]),
                 lambda: ops.rms_norm(x, g, residual=x, out=x, sum_out=x), lambda: ops.rms_norm(x, g.cpu()),
                 lambda: ops.rms_norm(x, g, out=torch.empty(8, 2, device=dev).t())):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ the product

def activate(y: torch.Tensor, act: str | None) -> torch.Tensor:
    if act == "gelu":
        return y * torch.special.ndtr(y)
    return y * torch.sigmoid(y) if act == "silu" else y


def dense_bound(a, w, k: int, t: torch.dtype) -> torch.Tensor:
    """The sum's error before its rounding to ``t``. The e4m3 instruction adds products eight at a time,
    each cut at 2^-13 of the eight's largest (at most seven are cut), the bf16 one within 24 bits;
    the eights' sums and the workgroup's parts are added in fp32, at most k / 8 + 20 of them, each
    addition cut or rounded at 2^-23 of the terms' sum."""
    terms = a.abs() @ w.abs().t()
    cut = 2.0 ** -13 if t != torch.float32 else 2.0 ** -23
    most = torch.zeros_like(terms)
    for j in range(0, k, 8):
        p = a[:, None, j:j + 8].abs() * w[None, :, j:j + 8].abs()
        most += p.amax(2)
    return 7 * cut * most + (k / 8 + 20) * 2.0 ** -23 * terms


def dense_case(pkg, dev, m, k, o, t, *, bias=False, residual=False, act=None, seed=0, loud=True):
    x = rand((m, k), seed + 1)
    if loud:
        x[:, ::17] *= 30
    x = pkg.ops.quantize8(x.to(dev))
    w = pkg.ops.quantize8((rand((o, k), seed + 2) / math.sqrt(k)).to(dev))
    b = rand((o,), seed + 3) if bias else None
    r = rand((m, o), seed + 4, t) if residual else None
    got = pkg.ops.dense8(x, w, None if b is None else b.to(dev), residual=None if r is None else r.to(dev), act=act,
                         dtype=t)
    assert got.dtype == t and got.shape == (m, o)
    a, ww = wide(x), wide(w)
    y = a @ ww.t()
    bound = dense_bound(a, ww, k, t)
    for extra in (b, r):
        if extra is not None:
            y = y + extra.double()
            bound = bound + 2.0 ** -23 * (y.abs() + extra.double().abs())
    # |gelu'|, |silu'| < 1.13; the activations themselves are evaluated to a few fp32 steps
    z = activate(y, act)
    err = (got.cpu().double() - z).abs()
    allowed = 1.13 * bound + z.abs() * (half_step(t) + 8 * 2.0 ** -23) + tiny(t) + (2.0 ** -23 * y.abs() if act else 0)
    assert (err <= allowed).all(), (err / allowed).max()
    return x, w, b, r, got


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize(("m", "k", "o"), [
    (1, 1, 1), (1, 128, 16), (1, 4096, 40), (2, 130, 17), (15, 640, 64), (16, 100, 33), (17, 768, 96), (33, 1000, 100),
    (64, 384, 129), (65, 512, 257), (77, 768, 512), (128, 129, 128), (130, 1152, 260), (257, 256, 300),
])
def test_dense8_matches_float64(pkg, dev, m, k, o, t) -> None:
    dense_case(pkg, dev, m, k, o, t)


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize(("m", "k", "o"), [(3, 300, 50), (70, 256, 130), (300, 200, 270)])
def test_dense8_epilogue(pkg, dev, m, k, o, act, t) -> None:
    dense_case(pkg, dev, m, k, o, t, bias=True, residual=True, act=act, seed=9)


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize(("m", "k", "o", "act"), [(3000, 100, 3100, None), (2561, 700, 4360, "gelu"), (4100, 256, 2999, "silu")])
def test_dense8_large(pkg, dev, m, k, o, act, t) -> None:
    """Sizes that the largest tiles serve, ragged in both directions, against float64 products on the
    device; the bound is the one above with the sum of the terms in the place of the eights' largest."""
    x = pkg.ops.quantize8(rand((m, k), 1).to(dev))
    w = pkg.ops.quantize8((rand((o, k), 2) / math.sqrt(k)).to(dev))
    b, r = rand((o,), 3).to(dev), rand((m, o), 4, t).to(dev)
    base = torch.full((m, o + 3), 7.0, dtype=t, device=dev)
    got = pkg.ops.dense8(x, w, b, residual=r, act=act, out=base[:, 2:2 + o], dtype=t)
    assert (base[:, :2] == 7).all() and (base[:, 2 + o:] == 7).all()
    a, ww = wide(x).to(dev), wide(w).to(dev)
    y = torch.mm(a, ww.t().contiguous()) + b.double() + r.double()
    terms = torch.mm(a.abs(), ww.abs().t().contiguous())
    bound = (7 * 2.0 ** (-13 if t != torch.float32 else -23) + (k / 8 + 20) * 2.0 ** -23) * terms
    bound += 2.0 ** -23 * (y.abs() + b.double().abs() + r.double().abs())
    z = activate(y, act)
    allowed = 1.13 * bound + z.abs() * (half_step(t) + 8 * 2.0 ** -23) + tiny(t) + (2.0 ** -23 * y.abs() if act else 0)
    err = (got.double() - z).abs()
    assert (err <= allowed).all(), (err / allowed).max()


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize(("m", "k", "o"), [
    (34, 2385, 552), (103, 1465, 5093), (600, 1300, 1100), (1301, 1123, 3148), (8000, 1250, 8100)])
def test_dense8_tiles(pkg, dev, m, k, o, t) -> None:
    """Long rows at sizes for every tile, blocks of very unlike scales: all rows of some outputs and all
    outputs of some rows, the last ones among them, against the bound of the small cases."""
    gen = torch.Generator().manual_seed(m)
    blocks = -(-k // 128)
    x, w = rand((m, k), 1), rand((o, k), 2)
    x *= torch.exp2(torch.randint(-6, 7, (m, blocks), generator=gen).float()).repeat_interleave(128, 1)[:, :k]
    w *= torch.exp2(torch.randint(-6, 7, (o, blocks), generator=gen).float()).repeat_interleave(128, 1)[:, :k]
    xq, wq = pkg.ops.quantize8(x.to(dev)), pkg.ops.quantize8(w.to(dev))
    got = pkg.ops.dense8(xq, wq, dtype=t).double()
    a, ww = wide(xq).to(dev), wide(wq).to(dev)
    rows = torch.cat((torch.randperm(m, generator=gen)[:40], torch.tensor([0, m - 1]))).to(dev)
    cols = torch.cat((torch.randperm(o, generator=gen)[:40], torch.tensor([0, o - 1]))).to(dev)
    for xs, ws, part in ((a, ww[cols], got[:, cols]), (a[rows], ww, got[rows])):
        y = torch.mm(xs, ws.t().contiguous())
        allowed = dense_bound(xs, ws, k, t)
        # Rounding to fp16 makes infinities of what is half a step (16) and more above its largest, 65504.
        top = 65520 if t == torch.float16 else math.inf
        inf = part.isinf()
        assert (y.abs() + allowed >= top)[inf].all() and (part[inf] * y[inf] > 0).all()
        assert (y.abs() - allowed < top)[~inf].all()
        allowed += y.abs() * half_step(t) + tiny(t)
        assert ((part - y).abs() <= allowed)[~inf].all(), ((part - y).abs() / allowed)[~inf].max()


# Sizes, ragged in both directions, for each kernel of dense8, whatever the result's type and the activation.
KERNELS = [(0, 45, 300, 71), (1, 673, 4507, 1435), (2, 165, 576, 7223), (3, 3619, 1700, 1735), (4, 6081, 4873, 8139)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize(("kernel", "m", "k", "o"), KERNELS)
def test_dense8_kernels_of_the_tested_sizes(pkg, kernel, m, k, o, t) -> None:
    """The sizes of test_dense8_of_every_kernel take the kernels that they are there for."""
    lib, kb = pkg._lib, -(-k // 128)
    for act in (0, 1, 2):
        a = lib.Dense8Args(rows=m, features=k, out_features=o, x_codes=16, x_pitch=kb * 128, x_scales=16,
                           x_scales_pitch=-(-kb // 4) * 4, w_codes=16, w_pitch=kb * 128, w_scales=16,
                           w_scales_pitch=-(-kb // 4) * 4, y=16, y_pitch=o, act=act, dtype=pkg.ops.ALL_DTYPES[t])
        assert lib.lib.ldx_dense8_kernel(ctypes.byref(a)) == kernel, act
    a.rows = 0
    refused(pkg, lib.lib.ldx_dense8_kernel(ctypes.byref(a)), "dense8")


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize(("kernel", "m", "k", "o"), KERNELS)
def test_dense8_of_every_kernel(pkg, dev, kernel, m, k, o, act, t) -> None:
    """Each kernel with a bias, a residual and an output that are column ranges at odd offsets, and an activation:
    all rows of some outputs and all outputs of some rows, the last ones among them, against the bound of the small
    cases; what stands beside the output stays."""
    g, gd = torch.Generator().manual_seed(k), torch.Generator(device=dev).manual_seed(k)
    x = pkg.ops.quantize8(torch.randn(m, k, generator=gd, device=dev))
    w = pkg.ops.quantize8(torch.randn(o, k, generator=gd, device=dev) / math.sqrt(k))
    b = torch.randn(o, generator=gd, device=dev)
    r = torch.randn(m, o + 4, generator=gd, device=dev).to(t)[:, 1:1 + o]
    base = torch.full((m, o + 3), 7.0, dtype=t, device=dev)
    got = pkg.ops.dense8(x, w, b, residual=r, act=act, out=base[:, 2:2 + o], dtype=t)
    assert (base[:, :2] == 7).all() and (base[:, 2 + o:] == 7).all()
    xs, ws = (q.codes.double().unflatten(-1, (-1, 128)) * q.scales.double()[:, :q.codes.shape[1] // 128, None] for q in (x, w))
    xs, ws = xs.flatten(1)[:, :k], ws.flatten(1)[:, :k]
    rows = torch.cat((torch.randperm(m, generator=g)[:20], torch.tensor([0, m - 1]))).to(dev)
    cols = torch.cat((torch.randperm(o, generator=g)[:20], torch.tensor([0, o - 1]))).to(dev)
    every = slice(None)
    for i, j in ((every, cols), (rows, every)):
        add = (b.double()[j], r.double()[i][:, j])
        y = torch.mm(xs[i], ws[j].t().contiguous())
        allowed = dense_bound(xs[i], ws[j], k, t)
        for extra in add:
            y = y + extra
            allowed = allowed + 2.0 ** -23 * (y.abs() + extra.abs())
        z = activate(y, act)
        allowed = 1.13 * allowed + z.abs() * (half_step(t) + 8 * 2.0 ** -23) + tiny(t) + (2.0 ** -23 * y.abs() if act else 0)
        err = (got.double()[i][:, j] - z).abs()
        assert (err <= allowed).all(), (err / allowed).max()


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [2, 700])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_dense8_activations_of_large_values(pkg, dev, act, m, t) -> None:
    """Values whose squares or exponentials leave fp32, infinities and NaN."""
    top = 6e4 if t == torch.float16 else 3e38
    b = torch.tensor([math.inf, NAN, top, -top, 1e4, -1e4, 90.0, -90.0, 0.0] * 40)
    x = pkg.ops.quantize8(torch.zeros(m, 130, device=dev))
    w = pkg.ops.quantize8(torch.ones(b.numel(), 130, device=dev))
    y = pkg.ops.dense8(x, w, b.to(dev), act=act, dtype=t).cpu()
    want = torch.tensor([math.inf, NAN, top, 0.0, 1e4, 0.0, 90.0, 0.0, 0.0] * 40).to(t)
    assert torch.equal(y.isnan(), want.isnan().expand(m, -1))
    assert torch.equal(y.nan_to_num(nan=1.0), want.nan_to_num(nan=1.0).expand(m, -1))


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [2, 700])
def test_dense8_silu_where_its_exponential_is_large(pkg, dev, m, t) -> None:
    """Down to where exp(-v) passes fp32 (v = -88.72); from -87.34 on 1 / (1 + exp(-v)) is below fp32's normal
    numbers. A few fp32 steps (as in dense_case) and the rounding to ``t``."""
    b = torch.tensor([-80.0, -87.0, -87.3, -87.4, -88.0, -88.5, -88.7, -1e-30, 3e-30] * 9)
    x = pkg.ops.quantize8(torch.zeros(m, 130, device=dev))
    w = pkg.ops.quantize8(torch.ones(b.numel(), 130, device=dev))
    y = pkg.ops.dense8(x, w, b.to(dev), act="silu", dtype=t).cpu().double()
    want = b.double() / (1 + torch.exp(-b.double()))
    assert ((y - want).abs() <= want.abs() * (half_step(t) + 8 * 2.0 ** -23) + tiny(t)).all(), y[0] / want


@gpu
@pytest.mark.parametrize("m", [4, 100, 600])
def test_dense8_scales_differ_by_block(pkg, dev, m) -> None:
    """Blocks of very unlike sizes, zero blocks and rows among them: each product takes its own scales."""
    k, o = 900, 70
    x, w = rand((m, k), 1), rand((o, k), 2)
    x *= torch.exp2(torch.randint(-20, 20, (m, 8), generator=torch.Generator().manual_seed(1)).float()).repeat_interleave(128, 1)[:, :k]
    w *= torch.exp2(-torch.randint(-20, 20, (o, 8), generator=torch.Generator().manual_seed(2)).float()).repeat_interleave(128, 1)[:, :k]
    x[0], x[:, 128:256], w[3] = 0, 0, 0
    xq, wq = pkg.ops.quantize8(x.to(dev)), pkg.ops.quantize8(w.to(dev))
    a, ww = wide(xq), wide(wq)
    for t in (torch.bfloat16, torch.float32):
        got = pkg.ops.dense8(xq, wq, dtype=t).cpu().double()
        y = a @ ww.t()
        assert ((got - y).abs() <= dense_bound(a, ww, k, t) + y.abs() * half_step(t) + tiny(t)).all()
        assert (got[0] == 0).all() and (got[:, 3] == 0).all()


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize(("m", "o"), [(3, 40), (150, 140), (1500, 700)])
def test_dense8_of_any_scale_byte(pkg, dev, m, o, t) -> None:
    """Bytes that quantize8 does not write: 0 (2^-127) and 254 are powers of two like the others, 255 is NaN for its
    row or output."""
    k = 300
    x, w = pkg.ops.quantize8(rand((m, k), 1).to(dev)), pkg.ops.quantize8(rand((o, k), 2).to(dev))
    xs, ws, xc, wc = (q.view(torch.uint8) for q in (x.scales, w.scales, x.codes, w.codes))
    xs[:, :3], ws[:, :3] = 120, 125
    # Small rows times large outputs; codes of at most 1 where the scale is 2^127 (bf16 has no larger number).
    one = torch.tensor(0x38, dtype=torch.uint8, device=dev)
    xs[0, :3], xs[1, :3], xs[2, 1] = 0, 3, 255
    wc[4:7] = torch.minimum(wc[4:7] & 0x7f, one)
    ws[4, :3], ws[5, :3], ws[6, :3], ws[7, 2] = 254, 240, 250, 255
    got = pkg.ops.dense8(x, w, dtype=t).cpu().double()
    a, ww = wide(x), wide(w)
    assert got[2].isnan().all() and got[:, 7].isnan().all()
    a[2], ww[7] = 0, 0
    y, terms = a @ ww.t(), a.abs() @ ww.abs().t()
    allowed = dense_bound(a, ww, k, t) + y.abs() * half_step(t) + tiny(t)
    if t == torch.float32:   # operands as bf16 values: those below 2^-126 to half of their last place, 2^-133
        allowed += 2.0 ** -134 * (ww.abs().sum(1) + a.abs().sum(1)[:, None])
    # Held to what stays in fp32 on the way and in t at the end.
    keep = (terms < 2.0 ** 127) & (y.abs() + allowed < (65504 if t == torch.float16 else 2.0 ** 127))
    keep[2], keep[:, 7] = False, False
    assert keep[:2].sum() > 70 and keep[:, 5].any() and ((got - y).abs() <= allowed)[keep].all(), ((got - y).abs() / allowed)[keep].max()


@gpu
def test_dense8_nan_stays_in_its_row_and_column(pkg, dev) -> None:
    for m, o in ((5, 40), (140, 150)):
        x, w = rand((m, 256), 1), rand((o, 256), 2)
        clean = pkg.ops.dense8(pkg.ops.quantize8(x.to(dev)), pkg.ops.quantize8(w.to(dev))).cpu()
        x[2, 9], w[7, 200] = NAN, math.inf
        y = pkg.ops.dense8(pkg.ops.quantize8(x.to(dev)), pkg.ops.quantize8(w.to(dev))).cpu()
        assert y[2].isnan().all() and y[:, 7].isnan().all()
        keep_r, keep_c = [i for i in range(m) if i != 2], [i for i in range(o) if i != 7]
        assert torch.equal(y[keep_r][:, keep_c], clean[keep_r][:, keep_c])


@gpu
@pytest.mark.parametrize("m", [3, 90, 520])
def test_dense8_leads_and_outputs(pkg, dev, m) -> None:
    """Leading axes, an output and a residual that are column ranges of wider tensors (odd offsets), the
    output over the residual."""
    k, o = 200, 72
    x = pkg.ops.quantize8(rand((2, m, k), 1).to(dev))
    w = pkg.ops.quantize8(rand((o, k), 2).to(dev))
    r = rand((2, m, o + 5), 3, torch.float16).to(dev)
    want = pkg.ops.dense8(x, w, residual=r[..., 3:3 + o].contiguous())
    assert want.shape == (2, m, o)
    base = torch.full((2, m, o + 9), 7.0, dtype=torch.float16, device=dev)
    out = base[..., 5:5 + o]
    assert pkg.ops.dense8(x, w, residual=r[..., 3:3 + o], out=out) is out
    assert torch.equal(out, want) and (base[..., :5] == 7).all() and (base[..., 5 + o:] == 7).all()
    z = r[..., 3:3 + o]
    pkg.ops.dense8(x, w, residual=z, out=z)
    assert torch.equal(z, want)


@gpu
def test_dense8_refuses_on_the_device(pkg, dev) -> None:
    ops = pkg.ops
    x, w = ops.quantize8(torch.ones(2, 200, device=dev)), ops.quantize8(torch.ones(3, 200, device=dev))
    for call in (lambda: ops.dense8(x, ops.quantize8(torch.ones(3, 100, device=dev))),
                 lambda: ops.dense8(x, w, act="relu"), lambda: ops.dense8(x, w, dtype=torch.float64),
                 lambda: ops.dense8(x, w, torch.ones(4, device=dev)), lambda: ops.dense8(x, w, torch.ones(1, 3, device=dev)),
                 lambda: ops.dense8(x, w, residual=torch.ones(2, 3, device=dev)),
                 lambda: ops.dense8(x, w, residual=torch.ones(2, 4, device=dev).half()),
                 lambda: ops.dense8(x, w, out=torch.empty(2, 3, device=dev)),
                 lambda: ops.dense8(x, w, out=torch.empty(3, 2, device=dev).half().t()),
                 lambda: ops.dense8(ops.Quantized8(x.codes, x.scales, 300), w),
                 lambda: ops.dense8(ops.Quantized8(x.codes[:1], x.scales, 200), w),
                 lambda: ops.dense8(x, ops.quantize8(torch.ones(1, 3, 200, device=dev)))):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ the cache

class Pages:
    """The cache in float64: appends and reads as the formulas say, page by page."""

    def __init__(self, cache):
        self.k = cache.k.cpu().double()
        self.v = cache.v.cpu().double().transpose(2, 3).contiguous()
        self.ks, self.vs = cache.k_scales.cpu().double(), cache.v_scales.cpu().double()

    def append(self, k, v, table, starts, counts=None):
        pages, heads = self.ks.shape
        for b, first in enumerate(starts.tolist()):
            n = k.shape[2] if counts is None else min(int(counts[b]), k.shape[2])
            if first < 0:
                continue
            for slot in range(first // 64, -(-(first + n) // 64)) if n > 0 else ():
                if slot >= table.shape[1] or not 0 <= int(table[b, slot]) < pages:
                    continue
                page = int(table[b, slot])
                lo, hi = max(first - 64 * slot, 0), min(first + n - 64 * slot, 64)
                for codes, scales, new in ((self.k, self.ks, k), (self.v, self.vs, v)):
                    put = new[b, :, 64 * slot + lo - first:64 * slot + hi - first].double()
                    to = scale_for(put.abs().nan_to_num(0.0, math.inf, math.inf).amax((1, 2)))
                    if lo:
                        to = torch.maximum(to, scales[page])
                        codes[page, :, :lo] = nearest8(codes[page, :, :lo] * (scales[page] / to)[:, None, None])
                    codes[page, :, lo:hi] = nearest8(put / to[:, None, None])
                    scales[page] = to

    def equals(self, cache):
        pairs = [(cache.k.cpu().double(), self.k), (cache.v.cpu().double().transpose(2, 3), self.v),
                 (cache.k_scales.cpu().double(), self.ks), (cache.v_scales.cpu().double(), self.vs)]
        for i, (got, want) in enumerate(pairs):
            assert torch.equal(got.nan_to_num(9999.0), want.nan_to_num(9999.0)), (i, (got != want).nonzero()[:4])

    def read(self, table_row, n):
        at = table_row[:-(-n // 64)].long()
        k = (self.k[at] * self.ks[at][..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
        v = (self.v[at] * self.vs[at][..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
        return k, v


def tables(b, width, spare=2, seed=0):
    return torch.randperm(b * width + spare, generator=torch.Generator().manual_seed(seed))[:b * width].reshape(b, width).int()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_append_token_by_token_and_in_parts(pkg, dev, d, t) -> None:
    """Lengths from one token on, page ends inside and between appends, scales that rise: codes and
    scales equal the float64 form's after every call, and pages in no table stay as they were."""
    heads, width = 2, 4
    cache = pkg.ops.Cache8.empty(3 * width + 2, heads, d, dev)
    for x in (cache.k, cache.v):
        x.view(torch.uint8).copy_(torch.randint(0, 256, x.shape, dtype=torch.uint8))
    ref, table = Pages(cache), tables(3, width)
    starts, parts = [0, 0, 0], [(1, None), (1, None), (63, [63, 1, 40]), (70, None), (5, [0, 5, 3]), (1, None), (64, [64, 20, 9])]
    for i, (n, counts) in enumerate(parts):
        k = rand((3, heads, n, d), 10 * i, t, 2.0 ** (i % 4 * 3 - 4))
        v = rand((3, heads, n, d), 10 * i + 1, t, 2.0 ** (i % 3 * 4 - 6))
        s, c = ints(*starts), None if counts is None else ints(*counts)
        ref.append(k, v, table, s, c)
        pkg.ops.cache8_append(cache, k.to(dev), v.to(dev), table.to(dev), s.to(dev),
                              counts=None if c is None else c.to(dev))
        ref.equals(cache)
        starts = [a + (n if counts is None else counts[j]) for j, a in enumerate(starts)]


@gpu
def test_append_leaves_out_what_it_cannot_place(pkg, dev) -> None:
    """Past the table, a negative start, pages that the cache does not have: nothing else changes."""
    cache = pkg.ops.Cache8.empty(8, 1, 32, dev)
    ref, table = Pages(cache), ints(0, 1, 2, 9, 3, -1, 4, 5).reshape(4, 2)
    k, v, starts = rand((4, 1, 100, 32), 1), rand((4, 1, 100, 32), 2), ints(60, 10, 20, -5)
    ref.append(k, v, table, starts)
    pkg.ops.cache8_append(cache, k.to(dev), v.to(dev), table.to(dev), starts.to(dev))
    ref.equals(cache)
    counts = ints(-3, 0, 7, 1000)
    starts = ints(0, 0, 0, 0)
    ref.append(k, v, table, starts, counts)
    pkg.ops.cache8_append(cache, k.to(dev), v.to(dev), table.to(dev), starts.to(dev), counts=counts.to(dev))
    ref.equals(cache)


@gpu
def test_append_of_nan_zero_and_strided_tokens(pkg, dev) -> None:
    cache = pkg.ops.Cache8.empty(4, 2, 64, dev)
    ref, table, starts = Pages(cache), tables(1, 2), ints(3)
    kv = rand((1, 70, 3, 2, 64), 5, torch.float16)          # interleaved projections
    kv[0, 4, 1, 0, 9] = NAN
    kv[0, 65:, 2] = 0
    k, v = kv[:, :, 1].transpose(1, 2), kv[:, :, 2].transpose(1, 2)
    ref.append(k, v, table, starts)
    kd = kv.to(dev)
    pkg.ops.cache8_append(cache, kd[:, :, 1].transpose(1, 2), kd[:, :, 2].transpose(1, 2), table.to(dev), starts.to(dev))
    ref.equals(cache)


@gpu
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("byte", [0, 1, 253, 254, 255])
def test_append_behind_tokens_of_any_scale(pkg, dev, d, byte) -> None:
    """A page that holds tokens under any E8M0 byte, also those that no append writes: the new ones are written
    under the larger scale; a page of NaN stays one, with its older codes."""
    old = torch.randint(0, 127, (2, 3, 2, 64, d), dtype=torch.uint8, generator=torch.Generator().manual_seed(d))
    for size in (0.0, 2.0 ** -126, 1.0, 3.0e38):
        cache = pkg.ops.Cache8.empty(3, 2, d, dev)
        cache.k.view(torch.uint8).copy_(old[0])
        cache.v.view(torch.uint8).copy_(old[1].transpose(2, 3))
        for s in (cache.k_scales, cache.v_scales):
            s.view(torch.uint8).fill_(byte)
        ref, table, starts = Pages(cache), ints(1).reshape(1, 1), ints(13)
        k, v = (rand((1, 2, 9, d), i).clamp(-1, 1) * size for i in (1, 2))
        ref.append(k, v, table, starts)
        pkg.ops.cache8_append(cache, k.to(dev), v.to(dev), table.to(dev), starts.to(dev))
        if byte < 255:
            ref.equals(cache)
            continue
        assert (cache.k_scales.view(torch.uint8)[1] == 255).all() and (cache.v_scales.view(torch.uint8)[1] == 255).all()
        assert torch.equal(cache.k.view(torch.uint8)[1, :, :13].cpu(), old[0, 1, :, :13])
        assert torch.equal(cache.v.view(torch.uint8)[1, :, :, :13].cpu(), old[1, 1, :, :13].transpose(1, 2))


def attention_reference(ref, q, table, lengths, scale, starts):
    """(result, error allowed before the rounding to q's type) in float64."""
    b, hq, lq, d = q.shape
    out, allowed = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    heads = ref.ks.shape[1]
    for i in range(b):
        n = int(lengths[i])
        if n <= 0:
            continue
        k, v = (x.repeat_interleave(hq // heads, 0) for x in ref.read(table[i], n))
        s = q[i].double() @ k.transpose(1, 2) * scale
        # fp32 scores: d products and sums, the scale, and the difference to the maximum
        off = (d + 6) * 2.0 ** -23 * ((q[i].double().abs() @ k.abs().transpose(1, 2)) * abs(scale)).amax(-1, keepdim=True)
        if starts is not None:
            pos = int(starts[i]) + torch.arange(lq)
            s = s.masked_fill(torch.arange(n) > pos[:, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
        seen = (p > 0) | (s > -math.inf)
        vz = torch.where(seen.any(1)[:, :, None], v, 0.0)
        l = p.sum(-1, keepdim=True)
        safe = torch.where(l > 0, l, 1.0)
        out[i] = p @ vz / safe
        mass = p @ vz.abs() / safe
        # Probabilities p rounded to fp16 are p (1 + e) + u, |e| <= 2^-11, |u| <= 2^-25 (below 2^-14). Both
        # sums of sum p v / sum p take the rounded ones: with o the exact result, the quotient is off by
        # sum (p e + u) (v - o) / sum p (1 + e), at most 2^-11 (mass + |o|) and 2^-25 (sum |v| + n |o|) / sum p,
        # times 1 + 2^-10 for the divisor. Scores are off by `off`, fp32 sums of n terms, the hardware's
        # exponential (2^-22).
        o = out[i].abs()
        under = 2.0 ** -25 * (seen.double() @ vz.abs() + seen.sum(-1, keepdim=True) * o) / safe
        allowed[i] = ((mass + o) * 2.0 ** -11 + under) * (1 + 2.0 ** -10) + mass * (2.2 * off + (n + 80) * 2.0 ** -23)
    return out, allowed


def filled(pkg, dev, b, heads, d, width, seed=0, lengths=None, spread=9):
    """A cache with codes everywhere (NaN codes behind the lengths), its float64 form and its table."""
    g = torch.Generator().manual_seed(seed)
    table = tables(b, width, seed=seed)
    cache = pkg.ops.Cache8.empty(b * width + 2, heads, d, dev)
    n = width * 64
    k, v = torch.randn(b, heads, n, d, generator=g), torch.randn(b, heads, n, d, generator=g)
    k *= torch.exp2(torch.randint(-2, 2, (b, heads, width, 1), generator=g).float()).repeat_interleave(64, 2)
    v *= torch.exp2(torch.randint(-spread, spread, (b, heads, width, 1), generator=g).float()).repeat_interleave(64, 2)
    pkg.ops.cache8_append(cache, k.to(dev), v.to(dev), table.to(dev), torch.zeros(b, dtype=torch.int32, device=dev))
    if lengths is not None:
        for i, n in enumerate(lengths.tolist()):
            for slot in range(max(n, 0) // 64, width):
                page, lo = int(table[i, slot]), max(n - 64 * slot, 0)
                cache.k.view(torch.uint8)[page, :, lo:] = 0x7f
                cache.v.view(torch.uint8)[page, :, :, lo:] = 0xff
    return cache, Pages(cache), table


# Columns of a page table with which 128 rows and more of one cache head share pages through LDS (the host
# decides by the table's width); a table that is longer than its sequences is what serving keeps anyway.
LONG = {64: 14000, 128: 2600, 256: 1300}


def longer(table: torch.Tensor, width: int | None) -> torch.Tensor:
    """``table`` followed by columns that name no page."""
    return table if width is None else torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1)


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_attention_kernels_of_the_tested_widths(pkg, d) -> None:
    """From 128 rows of a cache head on a table of LONG columns takes the kernel that shares pages, for any number of
    heads and sequences; fewer rows, the tests' short tables and heads of 32 the streaming one."""
    lib = pkg._lib

    def rows(batch, heads, group, q_len, width):
        a = lib.Cache8AttentionArgs(cache=_cache_args(lib, heads=heads, head_dim=d), batch=batch, q_heads=heads * group,
                                    q_len=q_len, q=16, o=16, scale=1.0, table=16, table_pitch=width, width=width, lengths=16)
        return lib.lib.ldx_cache8_attention_rows(ctypes.byref(a))

    for batch, heads, group, q_len in ((1, 1, 1, 128), (7, 1, 3, 50), (1, 1, 2, 70), (4, 2, 1, 150), (2, 2, 2, 100), (1, 1, 1, 300)):
        assert rows(batch, heads, group, q_len, LONG.get(d, 14000)) == (16 if d == 32 else 128)
        assert rows(1, heads, group, q_len, 8) == rows(batch, heads, group, 127 // group, LONG.get(d, 14000)) == 16
    assert rows(1, 3, 1, 0, 8) == lib.LDX_EINVAL


def attention_case(pkg, dev, t, b, heads, group, d, lq, lengths, starts, width, seed=0, scale=None, long=None, spread=9):
    scale = d ** -0.5 if scale is None else scale
    cache, ref, table = filled(pkg, dev, b, heads, d, width, seed, lengths, spread)
    q = rand((b, heads * group, lq, d), seed + 7, t)
    got = pkg.ops.cache8_attention(q.to(dev), cache, longer(table, long).to(dev), lengths.to(dev), scale,
                                   starts=None if starts is None else starts.to(dev))
    assert got.dtype == t and got.shape == q.shape
    want, allowed = attention_reference(ref, q, table, lengths, scale, starts)
    err = (got.cpu().double() - want).abs()
    bar = allowed * (1 + half_step(t)) + want.abs() * half_step(t) + tiny(t)
    assert (err <= bar).all(), ((err / bar).max(), (err > bar).nonzero()[:5])
    return got


@gpu
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize(("heads", "group", "lq"), [(1, 1, 1), (2, 4, 1), (3, 1, 5), (1, 8, 3), (2, 2, 40), (1, 3, 150)])
def test_attention_matches_float64(pkg, dev, heads, group, lq, d, t) -> None:
    """Lengths of none, one, page ends and their neighbours; NaN codes behind every length."""
    lengths = ints(0, 1, 63, 64, 65, 300, 448)
    attention_case(pkg, dev, t, 7, heads, group, d, lq, lengths, None, 7, seed=d + lq)


@gpu
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize(("heads", "group", "lq"), [(2, 4, 1), (1, 2, 7), (2, 1, 64), (1, 3, 131), (2, 4, 200)])
def test_attention_causal(pkg, dev, heads, group, lq, d, t) -> None:
    """Queries behind held tokens (none, some), with rows that see nothing (a start before 0) and a
    length below the last query's position."""
    starts = ints(0, 1, 100, -3, 250, 63)
    lengths = ints(lq, lq + 1, 100 + lq, lq, 250 + max(lq // 2, 1), 63 + lq)
    attention_case(pkg, dev, t, 6, heads, group, d, lq, lengths, starts, 8, seed=d + lq)


@gpu
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize(("heads", "group", "lq"), [(1, 1, 128), (2, 1, 129), (1, 3, 50), (2, 4, 65)])
def test_attention_of_many_rows(pkg, dev, heads, group, lq, d, t) -> None:
    """128 rows of a cache head and more: the last tile with one row, or full; lengths and starts as above."""
    attention_case(pkg, dev, t, 7, heads, group, d, lq, ints(0, 1, 63, 64, 65, 300, 448), None, 7, seed=d + lq, long=LONG[d])
    starts = ints(0, 1, 100, -3, 250, 63)
    lengths = ints(lq, lq + 1, 100 + lq, lq, 250 + max(lq // 2, 1), 63 + lq)
    attention_case(pkg, dev, t, 6, heads, group, d, lq, lengths, starts, 8, seed=d + lq, long=LONG[d])


@gpu
def test_cache_beyond_4_gib(pkg, dev) -> None:
    """Pages whose offsets pass 32 bits, written and read like the first ones."""
    heads, d, far, width = 4, 128, 140000, 20
    small, big = pkg.ops.Cache8.empty(width, heads, d, dev), pkg.ops.Cache8.empty(far, heads, d, dev)
    low = torch.arange(width, dtype=torch.int32, device=dev)[None]
    high = far - 1 - 7 * low
    k, v = rand((1, heads, 1200, d), 1).to(dev), rand((1, heads, 1200, d), 2).to(dev)
    for cache, table in ((small, low), (big, high)):
        pkg.ops.cache8_append(cache, k, v, table, ints(3).to(dev))
    for mine, theirs in zip((small.k, small.v, small.k_scales, small.v_scales), (big.k, big.v, big.k_scales, big.v_scales)):
        assert torch.equal(mine.view(torch.uint8), theirs.view(torch.uint8)[high[0].long()])
    for lq, long in ((1, None), (150, LONG[d])):
        q = rand((1, 8, lq, d), 3, torch.bfloat16).to(dev)
        n = ints(1203).to(dev)
        got = pkg.ops.cache8_attention(q, big, longer(high, long), n, 0.1)
        assert torch.equal(got, pkg.ops.cache8_attention(q, small, longer(low, long), n, 0.1))


@gpu
@pytest.mark.parametrize("d", [32, 64])
def test_attention_of_a_million_rows(pkg, dev, d) -> None:
    """More tiles of rows than a launch's second axis takes."""
    attention_case(pkg, dev, torch.bfloat16, 1, 1, 32, d, 33000, ints(70), None, 2)


@gpu
@pytest.mark.parametrize("lq", [1, 3, 200])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_attention_in_place(pkg, dev, d, lq) -> None:
    long = LONG.get(d) if lq > 100 else None
    cache, _, table = filled(pkg, dev, 2, 2, d, 30)
    q = rand((2, lq, 4, d), 3, torch.bfloat16).to(dev).transpose(1, 2)
    args = cache, longer(table, long).to(dev), ints(1900, 640).to(dev), 0.1
    want = pkg.ops.cache8_attention(q, *args)
    got = pkg.ops.cache8_attention(q, *args, out=q)
    assert got is q and torch.equal(got, want)


@gpu
@pytest.mark.parametrize("lq", [2, 140])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_value_scales_far_apart(pkg, dev, d, lq) -> None:
    """Pages of values up to 2^60 apart, in both orders."""
    long = LONG[d] if lq > 100 else None
    attention_case(pkg, dev, torch.bfloat16, 2, 1, 1, d, lq, ints(1000, 640), None, 16, long=long, spread=30)
    attention_case(pkg, dev, torch.bfloat16, 2, 1, 1, d, lq, ints(1000, 640), ints(1000 - lq, 500), 16, seed=5, long=long, spread=30)


@gpu
@pytest.mark.parametrize("lq", [3, 130])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_queries_before_a_page_do_not_feel_its_scale(pkg, dev, d, lq) -> None:
    """A page's scale, however large, or NaN, reaches only the queries that see the page."""
    long = LONG[d] if lq > 100 else None
    cache, _, table = filled(pkg, dev, 1, 2, d, 8)
    q = rand((1, 2, lq, d), 3, torch.bfloat16).to(dev)
    first = 256 - lq // 2   # half of the queries see page 4
    run = lambda: pkg.ops.cache8_attention(q, cache, longer(table, long).to(dev), ints(448).to(dev), 0.1, starts=ints(first).to(dev))
    want, page = run(), int(table[0, 4])
    assert want.isfinite().all()
    for scales in (cache.v_scales, cache.k_scales):
        was = scales.clone()
        for byte in (240, 255, 0):
            scales.view(torch.uint8)[page, 0] = byte
            got = run()
            assert torch.equal(got[:, 1], want[:, 1]) and torch.equal(got[:, 0, :256 - first], want[:, 0, :256 - first])
            seen = got[:, 0, 256 - first:]
            if byte == 255:
                assert seen.isnan().all()
            elif byte == 0 or scales is cache.v_scales:   # (keys of 448 * 2^113 and 64 channels of 4: scores pass fp32)
                assert not seen.isnan().any()
            if byte == 240 and scales is cache.v_scales:
                assert (seen.abs() > 2.0 ** 80).any()
        scales.copy_(was)
    assert torch.equal(run(), want)
    # A scale of NaN beside scales of 1, in a later page and in the first, which half of the queries do not see.
    cache.v_scales.view(torch.uint8).fill_(127)
    for page, first in ((int(table[0, 4]), first), (int(table[0, 0]), -(lq // 2))):
        want = run()
        cache.v_scales.view(torch.uint8)[page, 1] = 255
        got = run()
        cache.v_scales.view(torch.uint8)[page, 1] = 127
        at = lq // 2
        assert want.isfinite().all() and torch.equal(got[:, 0], want[:, 0]) and torch.equal(got[:, 1, :at], want[:, 1, :at])
        assert got[:, 1, at:].isnan().all()


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_of_many_rows_in_parts(pkg, dev, d) -> None:
    """Sequences of unequal lengths spread over several workgroups, some of which find nothing to do."""
    attention_case(pkg, dev, torch.float16, 3, 1, 2, d, 70, ints(5000, 700, 1), None, 80, long=LONG[d])
    attention_case(pkg, dev, torch.bfloat16, 3, 1, 1, d, 200, ints(5000, 700, 200), ints(4800, 500, 0), 80, long=LONG[d])


@gpu
@pytest.mark.parametrize(("b", "heads", "group", "d", "n"), [(2, 1, 2, 32, 9000), (1, 1, 1, 64, 20000), (2, 2, 8, 128, 9001), (1, 1, 4, 256, 5000)])
def test_attention_long(pkg, dev, b, heads, group, d, n) -> None:
    lengths = ints(*[n - 77 * i for i in range(b)])
    attention_case(pkg, dev, torch.float16, b, heads, group, d, 1, lengths, None, -(-n // 64) + 1)
    attention_case(pkg, dev, torch.bfloat16, b, heads, group, d, 3, lengths, lengths - 3, -(-n // 64) + 1)


@gpu
@pytest.mark.parametrize("lq", [1, 4, 100])
def test_attention_scores_far_apart(pkg, dev, lq) -> None:
    """Large scores: one key takes all, probabilities underflow, the running maximum rises often."""
    attention_case(pkg, dev, torch.float16, 2, 2, 2, 64, lq, ints(300, 129), None, 5, scale=3.0)
    attention_case(pkg, dev, torch.bfloat16, 2, 2, 2, 128, lq, ints(300, 129), ints(200, 100), 5, scale=-2.0)
    attention_case(pkg, dev, torch.float16, 2, 1, 2, 64, lq, ints(300, 129), None, 5, scale=0.0)
    if lq == 100:
        attention_case(pkg, dev, torch.float16, 2, 2, 2, 64, lq, ints(300, 129), None, 5, scale=3.0, long=LONG[64])
        attention_case(pkg, dev, torch.bfloat16, 2, 2, 2, 128, lq, ints(300, 129), ints(200, 100), 5, scale=-2.0, long=LONG[128])
        attention_case(pkg, dev, torch.float16, 2, 1, 2, 64, lq, ints(300, 129), None, 5, scale=0.0, long=LONG[64])


@gpu
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("lq", "d", "long"), [(1, 32, None), (3, 64, None), (20, 128, None), (2, 256, None), (130, 64, LONG[64]),
                                               (130, 128, LONG[128]), (130, 256, LONG[256])])
def test_attention_of_huge_scores(pkg, dev, lq, d, long, t) -> None:
    """Scores of 2^20 to 2^37, whose last place is up to 2^14: the key of the largest takes all, and no product's
    rounding carries its probability out of fp16."""
    n = 500
    cache = pkg.ops.Cache8.empty(10, 2, d, dev)
    table = tables(1, 8)
    k, v = rand((1, 2, n, d), 1, scale=100.0), rand((1, 2, n, d), 2)
    pkg.ops.cache8_append(cache, k.to(dev), v.to(dev), table.to(dev), ints(0).to(dev))
    kk, vv = Pages(cache).read(table[0], n)
    best = torch.randint(0, n, (lq,), generator=torch.Generator().manual_seed(3))
    q = torch.stack([kk[h, best] * 100 for h in range(2)])[None].to(t)    # towards one key each
    for scale in (2.0 ** -4, 1.0, 37.3, 1000.0):
        s = q[0].double() @ kk.transpose(1, 2) * scale
        off = (d + 6) * 2.0 ** -23 * (q[0].double().abs() @ kk.abs().transpose(1, 2) * scale).amax(-1)
        top = s.topk(2, -1)
        # The largest is ahead by more than fp32 scores are off, and by more than fp16 probabilities reach.
        assert (top.values[..., 0] - top.values[..., 1] > 2 * off + 40).all()
        want = torch.stack([vv[h, top.indices[h, :, 0]] for h in range(2)])
        got = pkg.ops.cache8_attention(q.to(dev), cache, longer(table, long).to(dev), ints(n).to(dev), scale).cpu().double()
        assert ((got[0] - want).abs() <= want.abs() * (half_step(t) + 2.0 ** -20) + tiny(t)).all(), scale


@gpu
@pytest.mark.parametrize("x", [15.3, 18.7, 20.5, 22.5, 23.6, 25.2])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize(("b", "n", "lq", "d", "long", "adds"), [
    (1, 100_000, 1, 64, None, 300), (600, 8_000, 1, 64, None, 300), (300, 8_000, 2, 128, None, 300), (600, 8_000, 1, 32, None, 300),
    (600, 4_000, 1, 256, None, 300), (1, 30_000, 130, 64, LONG[64], 2200), (1, 30_000, 130, 128, LONG[128], 2200),
    (1, 30_000, 130, 256, LONG[256], 2200)])
def test_attention_keeps_the_weight_of_a_long_tail(pkg, dev, b, n, lq, d, long, adds, first, x) -> None:
    """One key, the first or the last, that outweighs each of ``n`` others by 2^x; their values are 1, its own 0
    in half of the channels and -1 in the others."""
    width, at = -(-(n + 1) // 64), 0 if first else n
    cache = pkg.ops.Cache8.empty(width, 1, d, dev)
    k, v = torch.zeros(1, 1, n + 1, d), torch.ones(1, 1, n + 1, d)
    k[0, 0, at], v[0, 0, at, :d // 2], v[0, 0, at, d // 2:] = 16.0, 0.0, -1.0
    table = torch.arange(width, dtype=torch.int32)[None]
    pkg.ops.cache8_append(cache, k.to(dev), v.to(dev), table.to(dev), ints(0).to(dev))
    p = 2.0 ** -x
    l = 1 + n * p
    o = torch.tensor([n * p / l, (n * p - 1) / l]).double().repeat_interleave(d // 2)
    mass = torch.tensor([n * p / l, (n * p + 1) / l]).double().repeat_interleave(d // 2)
    # Probabilities are rounded to fp16 2^7 times as large, p (1 + e) + u, |e| <= 2^-11, |u| <= 2^-25 / 2^7 (see
    # attention_reference); the dominant one, a power of two, exactly. Exponents of at most 28 are off by 2^-23 of
    # their size and the exponential by 2^-22: 2^-18 in all. fp32 sums of at most `adds` additions in a row (a
    # product's sixteens, pages, waves and parts).
    off = n * (p * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -32) * (1 - o) / l * (1 + 2.0 ** -10)
    allowed = off + adds * 2.0 ** -24 * (mass + o.abs())
    for t in (torch.float16, torch.bfloat16):
        q = torch.ones(b, 1, lq, d, dtype=t, device=dev)
        got = pkg.ops.cache8_attention(q, cache, longer(table, long).expand(b, -1).contiguous().to(dev),
                                       torch.full((b,), n + 1, dtype=torch.int32, device=dev), x * math.log(2.0) / (16 * d))
        err = (got.cpu().double() - o).abs()
        bar = allowed * (1 + half_step(t)) + o.abs() * half_step(t) + tiny(t)
        assert (err <= bar).all(), (err / bar).amax((0, 1, 2))


@gpu
@pytest.mark.parametrize("byte", [0, 1, 2, 20])
@pytest.mark.parametrize(("lq", "d", "long"), [(1, 32, None), (2, 64, None), (3, 128, None), (1, 256, None), (150, 64, LONG[64]),
                                               (130, 128, LONG[128]), (130, 256, LONG[256])])
def test_attention_of_keys_at_the_least_scales(pkg, dev, lq, d, long, byte) -> None:
    """Keys near 2^-126 under any E8M0 byte and queries near bf16's other end, whose scores are ordinary."""
    cache, _, table = filled(pkg, dev, 1, 1, d, 3)
    g = torch.Generator().manual_seed(1)
    cache.k_scales.view(torch.uint8).fill_(byte)
    codes = torch.tensor([0x48, 0xc8, 0x38, 0xb8, 0x30, 0], dtype=torch.uint8)        # 4, -4, 1, -1, 0.5, 0
    cache.k.view(torch.uint8).copy_(codes[torch.randint(0, 6, cache.k.shape, generator=g)])
    q = ((torch.randint(0, 2, (1, 1, lq, d), generator=g) * 2.0 - 1) * 2.0 ** 117).to(torch.bfloat16)
    for scale in (2.0 ** -8, 0.4, 3.0):
        got = pkg.ops.cache8_attention(q.to(dev), cache, longer(table, long).to(dev), ints(190).to(dev), scale).cpu().double()
        want, allowed = attention_reference(Pages(cache), q, table, ints(190), scale, None)
        bar = allowed * (1 + half_step(q.dtype)) + want.abs() * half_step(q.dtype) + tiny(q.dtype)
        assert ((got - want).abs() <= bar).all(), (scale, ((got - want).abs() / bar).max())


@gpu
@pytest.mark.parametrize(("lq", "d", "long"), [(1, 64, None), (9, 64, None), (70, 128, None), (200, 64, LONG[64]),
                                               (130, 128, LONG[128]), (130, 256, LONG[256])])
def test_attention_loud_page_of_small_weight(pkg, dev, lq, d, long) -> None:
    """A page whose values are 2^30 times the others' but whose keys nobody attends to: the small values
    of the others come out as they are."""
    cache, _, table = filled(pkg, dev, 1, 1, d, 4, seed=3)
    q = torch.ones(1, 1, lq, d, dtype=torch.float16, device=dev)
    k, v = torch.zeros(1, 1, 256, d, device=dev), rand((1, 1, 256, d), 4).to(dev)
    k[:, :, 64:128] = -16.0
    v[:, :, 64:128] *= 2.0 ** 30
    pkg.ops.cache8_append(cache, k, v, table.to(dev), ints(0).to(dev))
    ref = Pages(cache)
    lengths = ints(256)
    got = pkg.ops.cache8_attention(q, cache, longer(table, long).to(dev), lengths.to(dev), 1.0).cpu().double()
    want, _ = attention_reference(ref, q.cpu(), table, lengths, 1.0, None)
    # equal probabilities of 1: their rounding is exact, the sums are fp32
    assert ((got - want).abs() <= want.abs() * half_step(torch.float16) + 300 * 2.0 ** -23 * 4).all()


@gpu
@pytest.mark.parametrize(("lq", "group", "d", "long"), [
    (4, 1, 64, None), (70, 1, 64, None), (33, 4, 128, None), (200, 1, 32, None), (100, 2, 256, None),
    (200, 1, 64, LONG[64]), (130, 2, 128, LONG[128]), (300, 1, 256, LONG[256])])
def test_attention_nan_in_tokens_that_a_query_does_not_see(pkg, dev, lq, group, d, long) -> None:
    """A NaN key and a NaN value: queries before them are untouched, queries from them on are NaN (in that
    channel, for a value)."""
    cache, _, table = filled(pkg, dev, 1, 1, d, 7, seed=1)
    q = rand((1, group, lq, d), 2, torch.float16).to(dev)
    args = (longer(table, long).to(dev), ints(100 + lq).to(dev), d ** -0.5)
    starts = ints(100).to(dev)
    clean = pkg.ops.cache8_attention(q, cache, *args, starts=starts)
    at = 100 + lq // 2
    page, slot = int(table[0, at // 64]), at % 64
    cache.v.view(torch.uint8)[page, 0, 5, slot] = 0x7f
    got = pkg.ops.cache8_attention(q, cache, *args, starts=starts)
    assert torch.equal(got[:, :, :lq // 2], clean[:, :, :lq // 2])
    assert got[:, :, lq // 2:, 5].isnan().all()
    rest = [i for i in range(d) if i != 5]
    assert torch.equal(got[..., rest], clean[..., rest])
    cache.v.view(torch.uint8)[page, 0, 5, slot] = 0
    cache.k.view(torch.uint8)[page, 0, slot, 3] = 0xff
    got = pkg.ops.cache8_attention(q, cache, *args, starts=starts)
    assert got[:, :, :lq // 2].isfinite().all() and got[:, :, lq // 2:].isnan().all()


@gpu
@pytest.mark.parametrize(("lq", "long"), [(1, None), (90, None), (150, LONG[64])])
def test_attention_says_when_a_page_or_a_length_is_wrong(pkg, dev, lq, long) -> None:
    cache, _, table = filled(pkg, dev, 4, 2, 64, 5, seed=1)
    q = rand((4, 2, lq, 64), 2, torch.float16).to(dev)
    lengths = ints(320, 320, 130, 320)
    good = pkg.ops.cache8_attention(q, cache, longer(table, long).to(dev), lengths.to(dev), 0.1)
    table[1, 3], table[2, 3], table[3, 1] = 1 << 30, -7, -1      # sequence 2 does not reach its bad page
    got = pkg.ops.cache8_attention(q, cache, longer(table, long).to(dev), lengths.to(dev), 0.1)
    assert torch.equal(got[[0, 2]], good[[0, 2]]) and got[[1, 3]].isnan().all()
    got = pkg.ops.cache8_attention(q, cache, longer(table, long).to(dev), ints(320, -4, (long or 5) * 64 + 1, 1 << 30).to(dev), 0.1)
    assert torch.equal(got[0], good[0]) and (got[1] == 0).all() and got[2:].isnan().all()


@gpu
@pytest.mark.parametrize(("lq", "width"), [(1, 9), (70, 9), (140, LONG[64])])
def test_attention_layouts(pkg, dev, lq, width) -> None:
    """Head-interleaved q and out, a table that is part of a wider one, out given."""
    cache, _, table = filled(pkg, dev, 2, 2, 64, 5, seed=1)
    q = rand((2, 4, lq, 64), 2, torch.bfloat16).to(dev)
    lengths = ints(300, 90).to(dev)
    want = pkg.ops.cache8_attention(q, cache, longer(table, width - 4).to(dev), lengths, 0.1)
    inter = q.transpose(1, 2).contiguous().transpose(1, 2)
    buf = torch.zeros(2, lq, 4, 64 + 3, dtype=torch.bfloat16, device=dev)
    out = buf[..., 1:65].transpose(1, 2)
    widetable = torch.full((2, width), -1, dtype=torch.int32)
    widetable[:, 2:7] = table
    got = pkg.ops.cache8_attention(inter, cache, widetable.to(dev)[:, 2:width - 2], lengths, 0.1, out=out)
    assert got is out and torch.equal(out, want)
    assert (buf[..., 0] == 0).all() and (buf[..., 65:] == 0).all()


@gpu
def test_cache_refuses_on_the_device(pkg, dev) -> None:
    ops = pkg.ops
    cache = ops.Cache8.empty(4, 2, 64, dev)
    q = torch.zeros(1, 2, 3, 64, dtype=torch.float16, device=dev)
    table, n = torch.zeros(1, 2, dtype=torch.int32, device=dev), ints(5).to(dev)
    bad_v = ops.Cache8(cache.k, cache.v[:, :1], cache.k_scales, cache.v_scales)
    for call in (lambda: ops.cache8_attention(q.float(), cache, table, n, 1.0),
                 lambda: ops.cache8_attention(q[:, :1], cache, table, n, 1.0),
                 lambda: ops.cache8_attention(q[..., :32], cache, table, n, 1.0),
                 lambda: ops.cache8_attention(q, cache, table.long(), n, 1.0),
                 lambda: ops.cache8_attention(q, cache, table[:, :0], n, 1.0),
                 lambda: ops.cache8_attention(q, cache, table, n.repeat(2), 1.0),
                 lambda: ops.cache8_attention(q, cache, table, n, NAN),
                 lambda: ops.cache8_attention(q, bad_v, table, n, 1.0),
                 lambda: ops.cache8_attention(q, cache, table, n, 1.0, out=q[:, :, :2]),
                 lambda: ops.cache8_attention(q, cache, table, n, 1.0, out=q[:, :, :1].expand(-1, -1, 3, -1)),
                 lambda: ops.cache8_attention(q, cache, table, n, 1.0, out=q.flatten().as_strided(q.shape, (384, 64, 64, 1))),
                 lambda: ops.cache8_attention(q, cache, table, n, 1.0, starts=n.cpu()),
                 lambda: ops.cache8_append(cache, q, q[:, :, :1], table, n),
                 lambda: ops.cache8_append(cache, q, q.float(), table, n),
                 lambda: ops.cache8_append(cache, q[:, :1], q[:, :1], table, n),
                 lambda: ops.cache8_append(cache, q, q, table, n, counts=n.long())):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ together

class Block:
    """A transformer block on the 8-bit operators: norm, fused projection, append, attention, output
    projection on the residual, norm, feed-forward."""

    def __init__(self, ops, dev, c, heads, kv, d, seed=0):
        self.ops, self.heads, self.kv, self.d = ops, heads, kv, d
        w = lambda o, i, s: ops.quantize8((rand((o, i), seed + s) / math.sqrt(i)).to(dev))
        self.qkv, self.o = w((heads + 2 * kv) * d, c, 1), w(c, heads * d, 2)
        self.up, self.down = w(2 * c, c, 3), w(c, 2 * c, 4)
        self.g1, self.g2 = (1 + rand((c,), seed + s, scale=0.1).to(dev) for s in (5, 6))

    def __call__(self, x, cache, table, starts, lengths):
        ops, (b, n, c) = self.ops, x.shape
        qkv = ops.dense8(ops.rms_norm(x, self.g1, quantize=True), self.qkv)
        q, k, v = qkv.unflatten(-1, (-1, self.d)).transpose(1, 2).split([self.heads, self.kv, self.kv], 1)
        ops.cache8_append(cache, k, v, table, starts)
        a = torch.empty(b, n, self.heads, self.d, dtype=x.dtype, device=x.device)
        ops.cache8_attention(q, cache, table, lengths, self.d ** -0.5, starts=starts, out=a.transpose(1, 2))
        y, x = ops.rms_norm(ops.dense8(ops.quantize8(a.flatten(2)), self.o), self.g2, residual=x, quantize=True)
        return ops.dense8(ops.quantize8(ops.dense8(y, self.up, act="gelu")), self.down, residual=x)


@gpu
def test_block_prompt_then_tokens_equals_all_at_once(pkg, dev) -> None:
    """A prompt and then token by token against the float64 formula over the same cache, step by step; the
    whole chain repeats bit for bit."""
    b, c, heads, kv, d, n = 2, 192, 6, 2, 32, 70
    block = Block(pkg.ops, dev, c, heads, kv, d)
    x = rand((b, n + 6, c), 9, torch.float16).to(dev)

    def go():
        cache = pkg.ops.Cache8.empty(2 * b + 1, kv, d, dev)
        table = tables(b, 2, spare=1).to(dev)
        outs, at = [], 0
        for step in [n] + [1] * 6:
            starts = torch.full((b,), at, dtype=torch.int32, device=dev)
            outs.append(block(x[:, at:at + step], cache, table, starts, starts + step))
            at += step
        return torch.cat(outs, 1), cache

    y, cache = go()
    y2, cache2 = go()
    assert torch.equal(y, y2) and torch.equal(cache.k.view(torch.uint8), cache2.k.view(torch.uint8))
    # float64 of the last step over the cache as it stands
    ref, at = Pages(cache), n + 5
    last = x[:, at:].cpu()
    qz = lambda z: (lambda cs: (cs[0].unflatten(-1, (-1, 128)) * cs[1][..., None]).flatten(-2)[..., :z.shape[-1]])(rows8(z))
    norm = lambda z, g: norm_reference(z, g.cpu(), 1e-6, None)[1]
    qkv = qz(norm(last, block.g1)) @ wide(block.qkv).t()
    q = qkv[..., :heads * d].half().unflatten(-1, (heads, d)).transpose(1, 2)
    a, _ = attention_reference(ref, q, tables(b, 2, spare=1), ints(at + 1, at + 1), d ** -0.5, None)
    mid = (last.double() + (qz(a.transpose(1, 2).flatten(2)) @ wide(block.o).t())).half()
    h = qz(norm(mid, block.g2)) @ wide(block.up).t()
    want = qz(activate(h, "gelu")) @ wide(block.down).t() + mid.double()
    # Values that lie next to a rounding border fall to either side in fp16 and in float64; an 8-bit step
    # of 2^-3 in single features of one of three quantized inputs moves a result by 2^-4 / sqrt(features)
    # of its size each. The whole is held to a relative 2-norm of 2^-6.
    rel = (y[:, -1:].cpu().double() - want).norm() / want.norm()
    assert rel < 2.0 ** -6, rel


@gpu
def test_captured_step_replays_with_new_inputs(pkg, dev) -> None:
    """One step captured: positions, lengths and tokens come from device memory, so each replay appends and
    attends at the next position, equal to the eager chain, with eager work between the replays."""
    b, c, heads, kv, d = 3, 128, 4, 2, 64
    block = Block(pkg.ops, dev, c, heads, kv, d, seed=3)
    table = tables(b, 40).to(dev)                       # wide enough for several workgroups a sequence
    x = rand((b, 140, c), 4, torch.float16).to(dev)
    caches = [pkg.ops.Cache8.empty(b * 40 + 2, kv, d, dev) for _ in range(2)]
    starts = torch.zeros(b, dtype=torch.int32, device=dev)
    for cache in caches:
        block(x[:, :130], cache, table, starts, starts + 130)
    token = x[:, 130:131].clone()
    pos = torch.full((b,), 130, dtype=torch.int32, device=dev)
    ends = pos + 1
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        block(token, caches[1], table, pos, ends)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(token, caches[1], table, pos, ends)
    for i in range(4):
        token.copy_(x[:, 130 + i:131 + i])
        pos.fill_(130 + i)
        ends.fill_(131 + i)
        graph.replay()
        torch.cuda.synchronize()
        now = torch.full((b,), 130 + i, dtype=torch.int32, device=dev)
        want = block(x[:, 130 + i:131 + i], caches[0], table, now, now + 1)
        assert torch.equal(y, want), i
        assert torch.equal(caches[0].v.view(torch.uint8), caches[1].v.view(torch.uint8))


@gpu
def test_two_streams_at_once(pkg, dev) -> None:
    """Calls on two streams share nothing: results equal those of one stream."""
    cases = []
    for seed in (1, 2):
        cache, _, table = filled(pkg, dev, 1, 1, 64, 60, seed=seed)
        q = rand((1, 4, 1, 64), seed, torch.float16).to(dev)
        x = pkg.ops.quantize8(rand((5, 2048), seed).to(dev))
        w = pkg.ops.quantize8(rand((64, 2048), seed + 5).to(dev))
        cases.append((q, cache, table.to(dev), ints(3800).to(dev), x, w))
    run = lambda c: (pkg.ops.cache8_attention(*c[:4], 0.1), pkg.ops.dense8(c[4], c[5]))
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(run(c))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
