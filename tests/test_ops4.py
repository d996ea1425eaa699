"""The rotation of heads and the 4-bit cache: append, read and attention. Refusals through the C ABI run on the
CPU; results are compared with float64 on an MI355X."""

from __future__ import annotations

import ctypes
import math
import subprocess

import pytest
import torch

from tests.conftest import REPO

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
HALF = [torch.float16, torch.bfloat16]
DIMS = [32, 64, 128, 256]
NAN = math.nan
VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def tiny(t: torch.dtype) -> float:
    """Half the spacing of ``t``'s subnormal numbers."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def rand(shape, seed, t=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(t)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def tables(b, width, spare=2, seed=0):
    return torch.randperm(b * width + spare, generator=torch.Generator().manual_seed(seed))[:b * width].reshape(b, width).int()


# ------------------------------------------------------------------ refusals on the CPU

def test_structs_match_c_layout(pkg, tmp_path) -> None:
    lib = pkg._lib
    fields = {"ldx_rotate_heads_args": lib.RotateHeadsArgs, "ldx_cache4": lib.Cache4Block,
              "ldx_cache4_append_args": lib.Cache4AppendArgs, "ldx_cache4_read_args": lib.Cache4ReadArgs,
              "ldx_cache4_attention_args": lib.Cache4AttentionArgs}
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "ldx.h"', "int main(void) {"]
    for cname, cls in fields.items():
        src.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        src += [f'printf("{cname} {f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in cls._fields_]
    src.append('printf("consts block4 %d\\nconsts page4 %d\\nconsts axes %d\\n", LDX_BLOCK4, LDX_PAGE4, LDX_ROTARY_AXES); return 0; }')
    (tmp_path / "l.c").write_text("\n".join(src))
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        cname, what, val = line.split()
        if cname == "consts":
            want = {"block4": lib.BLOCK4, "page4": lib.PAGE4, "axes": lib.ROTARY_AXES}[what]
        else:
            want = ctypes.sizeof(fields[cname]) if what == "size" else getattr(fields[cname], what).offset
        assert int(val) == want, line


def test_fillers_put_each_value_where_its_field_is(pkg) -> None:
    import ctypes
    flat = lambda v: [x for i in v for x in flat(i)] if isinstance(v, ctypes.Array) else \
        [x for name, _ in v._fields_ for x in flat(getattr(v, name))] if isinstance(v, ctypes.Structure) else [v]
    for kind in (pkg._lib.RotateHeadsArgs, pkg._lib.Cache4AppendArgs, pkg._lib.Cache4ReadArgs, pkg._lib.Cache4AttentionArgs):
        fill, values = pkg._lib.filler(kind), list(range(1, len(flat(kind())) + 1))
        assert flat(fill(*values)) == values
        for bad in (values[:-1], [*values, 1], [1 << 64, *values[1:]], [*values[:-1], None], [*values[:-1], 1.5]):
            with pytest.raises(ValueError, match=kind.__name__):
                fill(*bad)
    for scale in (1e300, "1"):
        values = list(range(1, len(flat(pkg._lib.Cache4AttentionArgs())) + 1))
        values[19] = scale
        with pytest.raises(ValueError, match="Cache4AttentionArgs"):
            pkg.ops._cache4_attention_args(*values)


def refused(pkg, rc: int, word: str) -> None:
    assert rc == pkg._lib.LDX_EINVAL
    assert word in pkg._lib.last_error(), pkg._lib.last_error()


@pytest.mark.parametrize("bad", [
    {"q": None}, {"q_out": None}, {"positions": None}, {"turns": None}, {"k": None}, {"k_out": None}, {"k_heads": -1},
    {"dtype": 3}, {"head_dim": 0}, {"head_dim": 33}, {"head_dim": 514}, {"q_heads": 0}, {"q_heads": 70000}, {"batch": 0},
    {"tokens": 0}, {"batch": 70000, "tokens": 70000}, {"axes": 0}, {"axes": 5}, {"axis_dims": (16, 20)}, {"axis_dims": (3, 4)},
    {"axis_dims": (0, 4)}, {"axis_dims": (-2, 4)},
    {"batch": 0x7fff, "tokens": 0xffff, "head_dim": 512}, {"q_gamma": 16, "eps": 0.0}, {"k_gamma": 16, "eps": NAN},
])
def test_rotate_heads_refuses(pkg, bad) -> None:
    a = pkg._lib.RotateHeadsArgs(batch=1, tokens=1, q_heads=1, k_heads=1, head_dim=32, dtype=0, q=16, q_out=16, k=16, k_out=16,
                                 axes=2, axis_dims=(16, 16), positions=16, turns=16, eps=1e-6)
    for k, v in bad.items():
        setattr(a, k, (ctypes.c_int32 * 4)(*v) if k == "axis_dims" else v)
    refused(pkg, pkg._lib.lib.ldx_rotate_heads(ctypes.byref(a), None), "rotate_heads")


def _cache_args(lib, **kw):
    c = dict(k=16, v=16, k_scales=16, v_scales=16, pages=2, heads=2, head_dim=64)
    c.update({k: v for k, v in kw.items() if k in c})
    return lib.Cache4Block(**c)


STORE_BAD = [{"pages": 0}, {"heads": 0}, {"heads": 9000}, {"head_dim": 48}, {"head_dim": 512}, {"k_scales": None}, {"k_scales": 8}, {"v": 24},
             {"tokens": 0}, {"tokens": (1 << 28) + 1}, {"batch": 0}, {"batch": 70000}, {"width": 0}, {"table_pitch": 0},
             {"table": None}, {"dtype": 9}, {"src": None}]


@pytest.mark.parametrize("bad", [*STORE_BAD, {"starts": None}])
def test_cache4_append_refuses(pkg, bad) -> None:
    lib = pkg._lib
    a = lib.Cache4AppendArgs(cache=_cache_args(lib, **bad), batch=1, tokens=1, k=16, v=16, table=16, table_pitch=1,
                             width=1, starts=16)
    for k, v in bad.items():
        if k == "src":
            a.v = v
        elif k not in ("k", "v") and hasattr(a, k):
            setattr(a, k, v)
    refused(pkg, lib.lib.ldx_cache4_append(ctypes.byref(a), None), "cache4_append")


@pytest.mark.parametrize("bad", [*STORE_BAD, {"lengths": None}])
def test_cache4_read_refuses(pkg, bad) -> None:
    lib = pkg._lib
    a = lib.Cache4ReadArgs(cache=_cache_args(lib, **bad), batch=1, tokens=1, k=16, v=16, table=16, table_pitch=1,
                           width=1, lengths=16)
    for k, v in bad.items():
        if k == "src":
            a.v = v
        elif k not in ("k", "v") and hasattr(a, k):
            setattr(a, k, v)
    refused(pkg, lib.lib.ldx_cache4_read(ctypes.byref(a), None), "cache4_read")


@pytest.mark.parametrize("bad", [
    {"pages": 0}, {"head_dim": 16}, {"q_heads": 3}, {"q_heads": 0}, {"q_len": 0}, {"batch": 0}, {"width": 0},
    {"width": 1 << 25, "table_pitch": 1 << 25}, {"table_pitch": 0}, {"lengths": None}, {"dtype": 1}, {"scale": NAN},
    {"scale": 1e31}, {"src": None}, {"q_len": 1 << 30}, {"q_len": 1 << 27},
])
def test_cache4_attention_refuses(pkg, bad) -> None:
    lib = pkg._lib
    a = lib.Cache4AttentionArgs(cache=_cache_args(lib, **bad), batch=1, q_heads=2, q_len=1, q=16, o=16, scale=1.0,
                                table=16, table_pitch=1, width=1, lengths=16)
    for k, v in bad.items():
        if k == "src":
            a.q = v
        elif hasattr(a, k):
            setattr(a, k, v)
    assert lib.lib.ldx_cache4_attention_workspace_bytes(ctypes.byref(a)) == 0
    refused(pkg, lib.lib.ldx_cache4_attention(ctypes.byref(a), None), "cache4_attention")


def test_attention_workspace_is_bounded(pkg) -> None:
    """Partial results are at most 256 MiB, whatever a call's size; long sequences of few queries are spread over
    workgroups, short ones are not."""
    lib = pkg._lib

    def parts(batch, heads, group, q_len, d, width):
        a = lib.Cache4AttentionArgs(cache=_cache_args(lib, heads=heads, head_dim=d), batch=batch, q_heads=heads * group,
                                    q_len=q_len, q=16, o=16, scale=1.0, table=16, table_pitch=width, width=width, lengths=16)
        n = lib.lib.ldx_cache4_attention_workspace_bytes(ctypes.byref(a))
        per = batch * heads * group * q_len * (d + 2) * 4
        assert n % per == 0 and n <= 256 << 20, (batch, heads, group, q_len, d, width, n)
        return max(n // per, 1)

    assert parts(1, 8, 1, 1, 128, 1024) > 1 and parts(1, 1, 1, 1, 64, 20000) > 1 and parts(1, 8, 1, 1, 64, 5) == 1
    gen = torch.Generator().manual_seed(1)
    log = lambda lo, hi: int(math.exp(math.log(lo) + torch.rand((), generator=gen).item() * math.log(hi / lo)))
    for _ in range(3000):
        d = DIMS[log(1, 16) % 4]
        batch, heads, group = log(1, 2000), log(1, 64), log(1, 16)
        parts(batch, heads, group, max(1, min(log(1, 100_000), 0x7fffffff // (batch * heads * group))), d, log(1, 1 << 24))


def test_cpu_tensors_are_refused(pkg) -> None:
    ops = pkg.ops
    x = torch.zeros(1, 1, 2, 32)
    cache = ops.Cache4.empty(2, 1, 32, device="cpu")
    one, at = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    rotary = ops.Rotary.make(32, device="cpu")
    for call in (lambda: ops.rotate_heads(x, x, at, rotary), lambda: ops.cache4_append(cache, x, x, at, one),
                 lambda: ops.cache4_read(cache, at, one, 3), lambda: ops.cache4_attention(x, cache, at, one, 1.0)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    for call in (lambda: ops.cache4_append(x, x, x, at, one), lambda: ops.cache4_read(x, at, one, 3),
                 lambda: ops.cache4_attention(x, x, at, one, 1.0)):
        with pytest.raises(ValueError, match="Cache4"):
            call()


def test_rotary_plan(pkg) -> None:
    make = pkg.ops.Rotary.make
    r = make((4, 6), theta=100.0, scale=(1.0, 0.5), device="cpu")
    want = [1.0, 100.0 ** -0.5, 0.5, 0.5 * 100.0 ** (-1 / 3), 0.5 * 100.0 ** (-2 / 3)]
    assert r.axes == (4, 6) and not r.interleaved
    assert torch.allclose(r.turns * 2 * math.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-15)
    assert make(8, device="cpu").axes == (8,)
    for bad in (lambda: make((3,), device="cpu"), lambda: make((), device="cpu"), lambda: make((4, 0), device="cpu"),
                lambda: make((4, 4), scale=(1.0,), device="cpu")):
        with pytest.raises(ValueError, match="axes"):
            bad()


def test_sizes_beyond_the_abi_fields_are_refused(pkg, monkeypatch) -> None:
    """Sizes that the C structs' 32 bits do not hold, none of which a call may take for the rest of them; tensors
    without memory stand in for those of a device."""
    ops = pkg.ops
    monkeypatch.setattr(ops, "_need", lambda *a: None)
    meta = lambda *shape, t=torch.float16: torch.empty(shape, dtype=t, device="meta")
    huge = (1 << 32) + 8
    ints32 = lambda *shape: meta(*shape, t=torch.int32)
    codes, scales = meta(2, 1, 64, 16, t=torch.uint8), meta(2, 1, 1, 64, t=torch.float8_e8m0fnu)
    cache = ops.Cache4(codes, codes, scales, scales)
    kv, many, one = meta(1, 1, 1, 32).expand(1, 1, huge, 32), meta(1, 1, 1, 32).expand(huge, 1, 1, 32), meta(1, 1, 1, 32)
    rotary = ops.Rotary(meta(16, t=torch.float64), (32,))
    with pytest.raises(ValueError, match="heads"):
        ops.rotate_heads(kv, None, ints32(1, 1).expand(1, huge), rotary, q_out=kv)
    with pytest.raises(ValueError, match="pages"):
        big = ops.Cache4(meta(1, 1, 64, 16, t=torch.uint8).expand(huge, 1, 64, 16), *[None] * 3)
        big.v, big.k_scales = big.k, meta(1, 1, 1, 64, t=torch.float8_e8m0fnu).expand(huge, 1, 1, 64)
        big.v_scales = big.k_scales
        monkeypatch.setattr(torch.Tensor, "is_contiguous", lambda self: True)
        ops.cache4_read(big, ints32(1, 1), ints32(1), 3)
    monkeypatch.undo()
    monkeypatch.setattr(ops, "_need", lambda *a: None)
    monkeypatch.setattr(ops, "_cache4_block", lambda c, what: ((16, 16, 16, 16, 2, 1, 32), 0))
    for word, call in (
            ("tokens", lambda: ops.cache4_append(cache, kv, kv, ints32(1, 1), ints32(1))),
            ("tokens", lambda: ops.cache4_append(cache, many, many, ints32(huge, 1), ints32(huge))),
            ("pages", lambda: ops.cache4_append(cache, one, one, ints32(1, huge), ints32(1))),
            ("tokens", lambda: ops.cache4_read(cache, ints32(1, 1), ints32(1), huge)),
            ("pages", lambda: ops.cache4_attention(one, cache, ints32(1, huge), ints32(1), 1.0)),
            ("queries", lambda: ops.cache4_attention(kv, cache, ints32(1, 1), ints32(1), 1.0, out=kv)),
            ("queries", lambda: ops.cache4_attention(many, cache, ints32(huge, 1), ints32(huge), 1.0, out=many))):
        with pytest.raises(ValueError, match=word):
            call()


# ------------------------------------------------------------------ rotation of heads

def rotated(x, gamma, eps, positions, rotary):
    """(result, size of each value's pair) in float64, pair by pair."""
    f = x.double()
    if gamma is not None:
        f = f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * gamma.double()
    y, size, at, p = f.clone(), f.abs(), 0, 0
    turns = rotary.turns.cpu()
    for axis, w in enumerate(rotary.axes):
        for i in range(w // 2):
            a, b = (at + 2 * i, at + 2 * i + 1) if rotary.interleaved else (at + i, at + i + w // 2)
            t = positions[axis].double() * turns[p]
            angle = (t - torch.round(t)) * (2 * math.pi)
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            y[..., a], y[..., b] = f[..., a] * c - f[..., b] * s, f[..., b] * c + f[..., a] * s
            size[..., a] = size[..., b] = torch.hypot(f[..., a], f[..., b])
            p += 1
        at += w
    return y, size


# Roundings in fp32, in units of 2^-24 of a pair's size: the squares' sum takes at most 16 of a lane and 6 of lanes, half
# of which reaches the root; mean and eps 3 halves, root 2, two products 2; cosine and sine 4 each of a turn's size
# (angle 1, the sums 3), sqrt(2) of both; the last two 2. 24 in all.
ROTATED = 24 * 2.0 ** -24


def check_rotated(got, x, gamma, eps, positions, rotary):
    want, size = rotated(x, gamma, eps, positions, rotary)
    t = x.dtype
    err = (got.cpu().double() - want).abs()
    bar = size * ROTATED * (1 + half_step(t)) + want.abs() * half_step(t) + tiny(t)
    assert (err <= bar).all(), ((err / bar).max(), (err > bar).nonzero()[:4])


ROTARIES = [((64,), 64), ((8, 12, 12), 32), ((16, 30, 30), 80), ((10, 6), 18), ((2,), 2), ((24, 24, 16), 72), ((32,), 128),
            ((256,), 256), ((2, 2, 2, 2), 14), ((128, 128, 256), 512), ((254, 6, 250), 512), ((252, 8, 240), 512)]


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("axes", "d"), ROTARIES)
def test_rotate_matches_float64(pkg, dev, axes, d, interleaved, t) -> None:
    """Sections whose halves divide by 8, 4, 2 and nothing; channels behind them; positions of both signs and large ones;
    with norms of both, of one and of none."""
    rotary = pkg.ops.Rotary.make(axes, interleaved=interleaved)
    q, k = rand((2, 3, 7, d), d, t, 2.0), rand((2, 2, 7, d), d + 1, t)
    g = torch.Generator().manual_seed(5)
    positions = torch.randint(-2000, 100_000, (len(axes), 2, 7), generator=g).int()
    positions[:, 0, 0], positions[0, 1, 3] = 0, 1_000_000_007
    qg, kg = 1 + rand((d,), 3, scale=0.2), rand((d,), 4)
    for a, b in ((qg, kg), (None, kg), (qg, None), (None, None)):
        on = lambda x: None if x is None else x.to(dev)
        yq, yk = pkg.ops.rotate_heads(q.to(dev), k.to(dev), positions.to(dev), rotary, q_gamma=on(a), k_gamma=on(b), eps=1e-5)
        check_rotated(yq, q, a, 1e-5, positions, rotary)
        check_rotated(yk, k, b, 1e-5, positions, rotary)
        assert yq.dtype == t and yq.transpose(1, 2).is_contiguous()
    alone = pkg.ops.rotate_heads(q.to(dev), None, positions.to(dev), rotary, q_gamma=qg.to(dev), eps=1e-5)
    check_rotated(alone, q, qg, 1e-5, positions, rotary)


@gpu
@pytest.mark.parametrize(("b", "l", "h", "kv", "d", "axes"), [
    (1, 1, 1, 1, 64, (64,)), (1, 1, 40, 8, 128, (128,)), (3, 1, 7, 1, 64, (32,)), (1, 5000, 2, 2, 32, (8, 12, 12)),
    (2, 1601, 5, 5, 80, (16, 30, 30)), (1, 3001, 1, 0, 64, (64,)), (65, 130, 3, 1, 6, (6,)), (1, 40, 200, 100, 256, (256,))])
def test_rotate_of_many_sizes(pkg, dev, b, l, h, kv, d, axes) -> None:
    """Calls of one token and of many, few heads and many, whose workgroups take one token or several."""
    rotary = pkg.ops.Rotary.make(axes)
    t = torch.bfloat16
    q, k = rand((b, h, l, d), 1, t), rand((b, kv, l, d), 2, t) if kv else None
    positions = torch.randint(0, 4000, (len(axes), b, l), generator=torch.Generator().manual_seed(1)).int()
    gamma = 1 + rand((d,), 3, scale=0.2)
    got = pkg.ops.rotate_heads(q.to(dev), None if k is None else k.to(dev), positions.to(dev), rotary, q_gamma=gamma.to(dev))
    check_rotated(got if k is None else got[0], q, gamma, 1e-6, positions, rotary)
    if k is not None:
        check_rotated(got[1], k, None, 1e-6, positions, rotary)


@gpu
@pytest.mark.parametrize("d", [32, 36, 64])
def test_rotate_layouts(pkg, dev, d) -> None:
    """Slices of one projection, (B, L, H, D) and (B, H, L, D) memory, odd offsets, positions expanded over the batch and
    (B, L) for one axis, in place and into given tensors that stand inside larger ones."""
    rotary = pkg.ops.Rotary.make(d)
    b, l, h, kv = 2, 9, 4, 2
    qkv = rand((b, l, h + 2 * kv, d), 1, torch.float16)
    at = torch.randint(0, 500, (1, l), generator=torch.Generator().manual_seed(1)).int()
    gamma = (1 + rand((d,), 3, scale=0.2)).to(dev)
    q, k = qkv[:, :, :h].transpose(1, 2), qkv[:, :, h:h + kv].transpose(1, 2)
    args = at.to(dev).expand(b, l), rotary
    want = pkg.ops.rotate_heads(q.contiguous().to(dev), k.contiguous().to(dev), *args, q_gamma=gamma, k_gamma=gamma)
    check_rotated(want[0], q, gamma.cpu(), 1e-6, at.expand(1, b, l), rotary)
    on = qkv.to(dev)
    sliced = lambda x: (x[:, :, :h].transpose(1, 2), x[:, :, h:h + kv].transpose(1, 2))
    got = pkg.ops.rotate_heads(*sliced(on), *args, q_gamma=gamma, k_gamma=gamma)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(on.cpu(), qkv)
    buf = torch.zeros(b, l, h + kv, d + 3, dtype=torch.float16, device=dev)
    outs = buf[:, :, :h, 1:d + 1].transpose(1, 2), buf[:, :, h:, 1:d + 1].transpose(1, 2)
    got = pkg.ops.rotate_heads(*sliced(on), *args, q_gamma=gamma, k_gamma=gamma, q_out=outs[0], k_out=outs[1])
    assert got[0] is outs[0] and torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    assert (buf[..., 0] == 0).all() and (buf[..., d + 1:] == 0).all()
    qi, ki = sliced(on)
    pkg.ops.rotate_heads(qi, ki, *args, q_gamma=gamma, k_gamma=gamma, q_out=qi, k_out=ki)
    assert torch.equal(qi, want[0]) and torch.equal(ki, want[1])
    assert torch.equal(on[:, :, h + kv:].cpu(), qkv[:, :, h + kv:])


@gpu
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
def test_rotate_of_extreme_heads(pkg, dev, t) -> None:
    """Squares past fp32 and below it, zeros; NaN and infinities stay in their head."""
    d = 64
    rotary = pkg.ops.Rotary.make(d)
    x = rand((1, 8, 1, d), 1).to(t)
    x[0, 1] *= 2.0 ** 100
    x[0, 2] *= 2.0 ** -80
    x[0, 3] = 0
    x[0, 4, 0, 5] = NAN
    x[0, 5, 0, 6] = math.inf
    x[0, 6] = 2.0 ** 126
    at, gamma = ints(3).reshape(1, 1, 1), torch.ones(d)
    got = pkg.ops.rotate_heads(x.to(dev), None, at.to(dev), rotary, q_gamma=gamma.to(dev), eps=1e-30).cpu()
    keep = [0, 1, 3, 6, 7]
    check_rotated(got[:, keep], x[:, keep], gamma, 1e-30, at, rotary)
    check_rotated(got[:, 2:3], x[:, 2:3], gamma, 1e-30, at, rotary)
    assert got[0, 4].isnan().all()
    assert got[0, 5, 0, [6, 38]].isnan().all()


@gpu
@pytest.mark.parametrize(("d", "axes"), [(128, (128,)), (36, (12, 10, 14))])
def test_rotate_beyond_4_gib(pkg, dev, d, axes) -> None:
    """Offsets past 32 bits, of values and of bytes: the last tokens are those of a call of their own."""
    ops, l, heads = pkg.ops, 70_001, 36 * 1024 // d
    rotary, gamma = ops.Rotary.make(axes, device=dev), torch.linspace(0.5, 2, d, device=dev)
    q = torch.zeros(1, l, heads, d, dtype=torch.float16, device=dev).transpose(1, 2)
    assert q.numel() > 2 ** 31
    tail = rand((1, heads, 40, d), 1, torch.float16).to(dev)
    q[:, :, -40:] = tail
    at = torch.arange(l, dtype=torch.int32, device=dev).expand(len(axes), 1, l)
    at = at[0] if len(axes) == 1 else at
    want = ops.rotate_heads(tail, None, at[..., -40:], rotary, q_gamma=gamma)
    got = ops.rotate_heads(q, None, at, rotary, q_gamma=gamma, q_out=q)
    assert got is q and torch.equal(got[:, :, -40:], want) and not got[:, :, :-40].any()


@gpu
def test_rotate_refuses_on_the_device(pkg, dev) -> None:
    ops = pkg.ops
    q = torch.zeros(1, 2, 3, 64, dtype=torch.float16, device=dev)
    at, rotary = torch.zeros(1, 3, dtype=torch.int32, device=dev), ops.Rotary.make(64)
    two = ops.Rotary.make((32, 32))
    for call in (lambda: ops.rotate_heads(q.double(), None, at, rotary), lambda: ops.rotate_heads(q[0], None, at, rotary),
                 lambda: ops.rotate_heads(q[:, :, :0], None, at[:, :0], rotary), lambda: ops.rotate_heads(q, q.float(), at, rotary),
                 lambda: ops.rotate_heads(q, q[:, :, :2], at, rotary), lambda: ops.rotate_heads(q, q[:, :0], at, rotary),
                 lambda: ops.rotate_heads(q, None, at.long(), rotary), lambda: ops.rotate_heads(q, None, at[:, :2], rotary),
                 lambda: ops.rotate_heads(q, None, at, two), lambda: ops.rotate_heads(q, None, at[None].expand(2, 1, 3).cpu(), two),
                 lambda: ops.rotate_heads(q, None, at, ops.Rotary.make(66)), lambda: ops.rotate_heads(q, None, at, rotary.turns),
                 lambda: ops.rotate_heads(q, None, at, ops.Rotary(rotary.turns.float(), (64,))),
                 lambda: ops.rotate_heads(q, None, at, ops.Rotary(rotary.turns[:-1], (64,))),
                 lambda: ops.rotate_heads(q, None, at, ops.Rotary.make((2,) * 5)),
                 lambda: ops.rotate_heads(q[..., ::2], None, at, ops.Rotary.make(32)),
                 lambda: ops.rotate_heads(q, None, at, rotary, q_gamma=torch.ones(63, device=dev)),
                 lambda: ops.rotate_heads(q, None, at, rotary, q_gamma=torch.ones(64)),
                 lambda: ops.rotate_heads(q, None, at, rotary, k_gamma=torch.ones(64, device=dev)),
                 lambda: ops.rotate_heads(q, None, at, rotary, q_gamma=torch.ones(64, device=dev), eps=0.0),
                 lambda: ops.rotate_heads(q, None, at, rotary, q_out=q[:, :1]),
                 lambda: ops.rotate_heads(q, None, at, rotary, q_out=q[:, :1].expand(1, 2, 3, 64)),
                 lambda: ops.rotate_heads(q, q, at, rotary, q_out=q, k_out=q),
                 lambda: ops.rotate_heads(q, q, at, rotary, q_out=q),
                 lambda: ops.rotate_heads(q, q.clone(), at, rotary, k_out=q),
                 lambda: ops.rotate_heads(q, None, at, rotary, q_out=q.view(1, 3, 2, 64).transpose(1, 2)),
                 lambda: ops.rotate_heads(q.clone(), q, at, rotary, k_out=q.view(1, 3, 2, 64).transpose(1, 2))):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ the cache

def scale4(amax: torch.Tensor) -> torch.Tensor:
    """The least 2^e, -126 <= e <= 125, with amax <= 6 * 2^e; 1 for zeros."""
    m, e = torch.frexp(amax)                      # amax = m 2^e, 0.5 <= m < 1; 6 = 0.75 * 2^3
    e = torch.where(m > 0.75, e - 2, e - 3).clamp(-126, 125)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), 1.0)


def nearest4(v: torch.Tensor) -> torch.Tensor:
    """The e2m1 value nearest to each ``v``, ties to the even code, magnitudes past 6 as 6; the sign stays."""
    a = v.abs().clamp(max=6.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=1.0))) - 1)
    return torch.copysign(torch.round(a / step) * step, v)


def rows4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(code values, scales) of float64 (..., D), NaN scales for blocks that are not finite."""
    y = x.double().unflatten(-1, (-1, 32))
    fine = y.isfinite().all(-1)
    y = torch.where(fine[..., None], y, 0.0)
    s = scale4(y.abs().amax(-1))
    return nearest4(y / s[..., None]).flatten(-2), torch.where(fine, s, NAN)


def unpacked(codes: torch.Tensor) -> torch.Tensor:
    c = codes.cpu().long()
    both = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    return torch.copysign(VALUES[both & 7], torch.where(both > 7, -1.0, 1.0).double())


class Pages:
    """The cache in float64: (pages, heads, 64, D) code values and (pages, heads, 64, D / 32) scales."""

    def __init__(self, cache):
        self.codes = [unpacked(x) for x in (cache.k, cache.v)]
        self.scales = [x.cpu().double().transpose(2, 3).contiguous() for x in (cache.k_scales, cache.v_scales)]

    def append(self, k, v, table, starts, counts=None):
        pages = self.codes[0].shape[0]
        for b, first in enumerate(starts.tolist()):
            n = k.shape[2] if counts is None else min(int(counts[b]), k.shape[2])
            for i in range(n if first >= 0 else 0):
                slot = (first + i) // 64
                if slot >= table.shape[1] or not 0 <= int(table[b, slot]) < pages:
                    continue
                page = int(table[b, slot])
                for codes, scales, new in zip(self.codes, self.scales, (k, v)):
                    codes[page, :, (first + i) % 64], scales[page, :, (first + i) % 64] = rows4(new[b, :, i])

    def equals(self, cache):
        now = Pages(cache)
        for mine, theirs in zip(self.codes + self.scales, now.codes + now.scales):
            assert torch.equal(mine.nan_to_num(9999.0), theirs.nan_to_num(9999.0)), (mine != theirs).nonzero()[:4]
        for mine, theirs in zip(self.codes, now.codes):
            assert torch.equal(torch.signbit(mine), torch.signbit(theirs))

    def values(self, which):
        return (self.codes[which].unflatten(-1, (-1, 32)) * self.scales[which][..., None]).flatten(-2)

    def read(self, table_row, n):
        at = table_row[:-(-n // 64)].long()
        return tuple((self.codes[w][at].unflatten(-1, (-1, 32)) * self.scales[w][at][..., None]).flatten(-2)
                     .transpose(0, 1).flatten(1, 2)[:, :n] for w in range(2))


def scramble(cache):
    """Any codes and scales from 2^-20 to 2^20."""
    g = torch.Generator().manual_seed(11)
    for x in (cache.k, cache.v):
        x.copy_(torch.randint(0, 256, x.shape, dtype=torch.uint8, generator=g))
    for x in (cache.k_scales, cache.v_scales):
        x.view(torch.uint8).copy_(torch.randint(107, 148, x.shape, dtype=torch.uint8, generator=g))


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", DIMS)
def test_append_token_by_token_and_in_parts(pkg, dev, d, t) -> None:
    """Lengths from one token on, page ends inside and between appends: codes and scales equal the float64 form's after
    every call, and other tokens stay as they were."""
    heads, width = 2, 4
    cache = pkg.ops.Cache4.empty(3 * width + 2, heads, d, dev)
    scramble(cache)
    ref, table = Pages(cache), tables(3, width)
    starts, parts = [0, 0, 0], [(1, None), (1, None), (63, [63, 1, 40]), (70, None), (5, [0, 5, 3]), (1, None), (64, [64, 20, 9])]
    for i, (n, counts) in enumerate(parts):
        k = rand((3, heads, n, d), 10 * i, t, 2.0 ** (i % 4 * 3 - 4))
        v = rand((3, heads, n, d), 10 * i + 1, t, 2.0 ** (i % 3 * 4 - 6))
        s, c = ints(*starts), None if counts is None else ints(*counts)
        ref.append(k, v, table, s, c)
        pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), s.to(dev),
                              counts=None if c is None else c.to(dev))
        ref.equals(cache)
        starts = [a + (n if counts is None else counts[j]) for j, a in enumerate(starts)]


@gpu
@pytest.mark.parametrize(("b", "heads", "n", "d"), [(1, 1, 1, 32), (48, 8, 1, 128), (1, 40, 1, 256), (2, 3, 1000, 64), (700, 2, 2, 32)])
def test_append_of_many_sizes(pkg, dev, b, heads, n, d) -> None:
    width = -(-(n + 40) // 64)
    cache = pkg.ops.Cache4.empty(b * width + 2, heads, d, dev)
    ref, table = Pages(cache), tables(b, width)
    starts = torch.randint(0, 40, (b,), generator=torch.Generator().manual_seed(1)).int()
    k, v = rand((b, heads, n, d), 1, torch.bfloat16), rand((b, heads, n, d), 2, torch.bfloat16)
    ref.append(k, v, table, starts)
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), starts.to(dev))
    ref.equals(cache)


@gpu
def test_append_leaves_out_what_it_cannot_place(pkg, dev) -> None:
    """Past the table, a negative start, pages that the cache does not have: nothing else changes."""
    cache = pkg.ops.Cache4.empty(8, 1, 32, dev)
    scramble(cache)
    ref, table = Pages(cache), ints(0, 1, 2, 9, 3, -1, 4, 5).reshape(4, 2)
    k, v, starts = rand((4, 1, 100, 32), 1), rand((4, 1, 100, 32), 2), ints(60, 10, 20, -5)
    ref.append(k, v, table, starts)
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), starts.to(dev))
    ref.equals(cache)
    starts, counts = ints(0, 0, 0, 2 ** 31 - 30), ints(-3, 0, 7, 1000)
    ref.append(k, v, table, starts, counts)
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), starts.to(dev), counts=counts.to(dev))
    ref.equals(cache)


@gpu
def test_append_shares_a_page_by_tokens(pkg, dev) -> None:
    """Two sequences that write different tokens of one page in one call."""
    cache = pkg.ops.Cache4.empty(2, 2, 64, dev)
    scramble(cache)
    ref, table, starts = Pages(cache), ints(1, 1).reshape(2, 1), ints(3, 30)
    k, v = rand((2, 2, 27, 64), 1), rand((2, 2, 27, 64), 2)
    ref.append(k, v, table, starts)
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), starts.to(dev))
    ref.equals(cache)


@gpu
@pytest.mark.parametrize("t", TYPES)
def test_append_of_special_and_strided_tokens(pkg, dev, t) -> None:
    """Interleaved projections at an odd offset with zeros of both signs, ties, the types' ends, NaN and infinities."""
    cache = pkg.ops.Cache4.empty(4, 2, 64, dev)
    ref, table, starts = Pages(cache), tables(1, 2), ints(3)
    buf = rand((1, 70, 3, 2, 67), 5, t)
    kv = buf[..., 1:65]
    info = torch.finfo(t)
    kv[0, 4, 1, 0, 9] = NAN
    kv[0, 5, 2, 1, 40] = -math.inf
    kv[0, 65:, 2] = 0
    kv[0, 66, 2, :, ::3] = -0.0
    kv[0, 6, 1, 0] = torch.linspace(-6, 6, 64)                                  # scale 1, ties among them
    kv[0, 7, 1, 0, :32] = torch.arange(32) * 0.25 - 2.0
    kv[0, 8, 1, 0, :32] = torch.arange(32) * (info.max / 31)
    kv[0, 9, 1, 0, :32] = torch.arange(32) * (info.smallest_normal * info.eps)  # subnormal numbers
    kv[0, 10, 1, 0, 32:] = info.smallest_normal * torch.linspace(-1, 7, 32)
    kv[0, 11, 1, 0, :32] = torch.linspace(-1, 1, 32) * 0.75
    kv[0, 11, 1, 0, 0] = -(0.75 + 0.75 * info.eps)                              # a neighbour of 6 * 2^-3
    kv[0, 12, 1, 1, 1:] = 0
    k, v = kv[:, :, 1].transpose(1, 2), kv[:, :, 2].transpose(1, 2)
    ref.append(k, v, table, starts)
    kd = buf.to(dev)[..., 1:65]
    pkg.ops.cache4_append(cache, kd[:, :, 1].transpose(1, 2), kd[:, :, 2].transpose(1, 2), table.to(dev), starts.to(dev))
    ref.equals(cache)
    for x, scales in ((k, ref.scales[0]), (v, ref.scales[1])):
        odd = (~x.isfinite()).unflatten(-1, (2, 32)).any(-1).sum()
        assert 1 <= odd <= 2 and scales.isnan().sum() == odd


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", DIMS)
def test_read_is_what_the_cache_holds(pkg, dev, d, t) -> None:
    """Every code under any scale byte, rounded to the type; lengths of none, one and page ends; rows behind a length are
    zeros, or as they were."""
    b, heads, width, n = 6, 2, 5, 300
    cache = pkg.ops.Cache4.empty(b * width + 2, heads, d, dev)
    scramble(cache)
    for x in (cache.k_scales, cache.v_scales):
        x.view(torch.uint8).copy_(torch.randint(0, 256, x.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(2)))
    ref, table = Pages(cache), tables(b, width)
    for starts in (None, ints(0, 5, 63, 64, -70, 250)):
        lengths = ints(0, 1, 64, 127, 300, 320)
        want = torch.zeros(2, b, heads, n, d, dtype=torch.float64)
        held = torch.zeros(b, n, dtype=torch.bool)
        for i in range(b):
            s, m = 0 if starts is None else int(starts[i]), int(lengths[i])
            full = torch.stack([x for x in ref.read(table[i], 320)])
            rows = torch.arange(max(s, 0), max(min(m, s + n), max(s, 0)))
            want[:, i, :, rows - s] = full[:, :, rows]
            held[i, rows - s] = True
        want = want.to(t)
        args = cache, table.to(dev), lengths.to(dev), n
        kw = dict(starts=None if starts is None else starts.to(dev), dtype=t)
        got = pkg.ops.cache4_read(*args, **kw)
        for w in range(2):
            assert torch.equal(got[w].cpu().nan_to_num(7.0), want[w].nan_to_num(7.0))
        buf = torch.full((2, b, n, heads, d + 5), 3.0, dtype=t, device=dev)
        out = buf[0, ..., 2:d + 2].transpose(1, 2), buf[1, ..., 2:d + 2].transpose(1, 2)
        same = pkg.ops.cache4_read(*args, **kw, out=out)
        assert same[0] is out[0] and same[1] is out[1]
        for w in range(2):
            kept = torch.where(held[:, None, :, None], want[w], torch.tensor(3.0, dtype=t))
            assert torch.equal(out[w].cpu().nan_to_num(7.0), kept.nan_to_num(7.0))
        assert (buf[..., :2] == 3).all() and (buf[..., d + 2:] == 3).all()


@gpu
def test_read_says_when_a_page_is_wrong(pkg, dev) -> None:
    cache = pkg.ops.Cache4.empty(6, 1, 64, dev)
    table, lengths = ints(0, 1, 9, 2, -1, 3).reshape(2, 3), ints(192, 300)
    k, v = pkg.ops.cache4_read(cache, table.to(dev), lengths.to(dev), 320)
    for x in (k.cpu(), v.cpu()):
        assert (x[0, :, :128] == 0).all() and x[0, :, 128:192].isnan().all() and (x[0, :, 192:] == 0).all()
        assert (x[1, :, :64] == 0).all() and x[1, :, 64:128].isnan().all() and (x[1, :, 128:192] == 0).all()
        assert x[1, :, 192:300].isnan().all() and (x[1, :, 300:] == 0).all()      # past the table


# ------------------------------------------------------------------ attention

# Columns of a page table with which 128 rows and more of one cache head share pages through LDS (the host decides by
# the table's width); a table that is longer than its sequences is what serving keeps anyway.
LONG = 5000


def longer(table: torch.Tensor, width: int | None) -> torch.Tensor:
    """``table`` followed by columns that name no page."""
    return table if width is None else torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1)


@pytest.mark.parametrize("d", DIMS)
def test_attention_kernels_of_the_tested_widths(pkg, d) -> None:
    """From 128 rows of a cache head on a table of LONG columns takes the kernel that shares pages, for any number of
    heads and sequences; fewer rows and the tests' short tables the streaming one."""
    lib = pkg._lib

    def rows(batch, heads, group, q_len, width):
        a = lib.Cache4AttentionArgs(cache=_cache_args(lib, heads=heads, head_dim=d), batch=batch, q_heads=heads * group,
                                    q_len=q_len, q=16, o=16, scale=1.0, table=16, table_pitch=width, width=width, lengths=16)
        return lib.lib.ldx_cache4_attention_rows(ctypes.byref(a))

    for batch, heads, group, q_len in ((1, 1, 1, 128), (7, 1, 3, 50), (1, 1, 2, 70), (4, 2, 1, 150), (2, 2, 2, 100), (1, 1, 1, 300)):
        assert rows(batch, heads, group, q_len, LONG) == 128
        assert rows(1, heads, group, q_len, 8) == rows(batch, heads, group, 127 // group, LONG) == 16
    assert rows(1, 3, 1, 0, 8) == lib.LDX_EINVAL


def attention_reference(ref, q, table, lengths, scale, starts, shared=False):
    """(result, error allowed before the rounding to q's type) in float64."""
    b, hq, lq, d = q.shape
    out, allowed = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    heads = ref.codes[0].shape[1]
    for i in range(b):
        n = int(lengths[i])
        if n <= 0:
            continue
        k, v = (x.repeat_interleave(hq // heads, 0) for x in ref.read(table[i], n))
        s = q[i].double() @ k.transpose(1, 2) * scale
        # fp32 scores: d products and sums (twice for a query in two parts), the scale, the difference to the reference
        off = (2 * d + 6) * 2.0 ** -24 * ((q[i].double().abs() @ k.abs().transpose(1, 2)) * abs(scale)).amax(-1, keepdim=True)
        if starts is not None:
            pos = int(starts[i]) + torch.arange(lq)
            s = s.masked_fill(torch.arange(n) > pos[:, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
        seen = s > -math.inf
        vz = torch.where(seen.any(1)[:, :, None], v, 0.0)
        l = p.sum(-1, keepdim=True)
        safe = torch.where(l > 0, l, 1.0)
        out[i] = p @ vz / safe
        mass = p @ vz.abs() / safe
        # A probability enters the values' product with 16 bits and their sum whole: 2^-16 of the mass. Where pages are
        # shared it is rounded to fp16 in both sums, p (1 + e) + u, |e| <= 2^-11, |u| <= 2^-32 of the largest: with o the
        # exact result the quotient is off by sum (p e + u) (v - o) / sum p (1 + e), at most 2^-11 (mass + |o|) and 2^-32
        # (sum |v| + n |o|) / sum p, times 1 + 2^-10 for the divisor. Scores are off by `off`; fp32 sums of n terms on
        # both sides; the hardware's exponential (2^-22). One below fp32's normal numbers, 2^-126 of the largest, is 0: of
        # a result of 1e-39 beside a dominant value of 0 that is a part.
        o = out[i].abs()
        least = (seen.double() @ vz.abs() + seen.sum(-1, keepdim=True) * o) / safe
        rounded = ((mass + o) * 2.0 ** -11 + 2.0 ** -32 * least) * (1 + 2.0 ** -10) if shared else mass * 2.0 ** -16
        allowed[i] = rounded + mass * (2.2 * off) + (mass + o) * (n + 40) * 2.0 ** -23 + 2.0 ** -126 * least
    return out, allowed


def filled(pkg, dev, b, heads, d, width, seed=0, lengths=None, spread=9):
    """A cache with codes everywhere (NaN scales behind the lengths), its float64 form and its table."""
    g = torch.Generator().manual_seed(seed)
    table = tables(b, width, seed=seed)
    cache = pkg.ops.Cache4.empty(b * width + 2, heads, d, dev)
    n = width * 64
    k, v = torch.randn(b, heads, n, d, generator=g), torch.randn(b, heads, n, d, generator=g)
    k *= torch.exp2(torch.randint(-2, 2, (b, heads, width, 1), generator=g).float()).repeat_interleave(64, 2)
    v *= torch.exp2(torch.randint(-spread, spread, (b, heads, width, 1), generator=g).float()).repeat_interleave(64, 2)
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), torch.zeros(b, dtype=torch.int32, device=dev))
    if lengths is not None:
        for i, n in enumerate(lengths.tolist()):
            for slot in range(max(n, 0) // 64, width):
                page, lo = int(table[i, slot]), max(n - 64 * slot, 0)
                for s in (cache.k_scales, cache.v_scales):
                    s.view(torch.uint8)[page, :, :, lo:] = 255
    return cache, Pages(cache), table


def agree(got, want, allowed):
    """``got`` is ``want`` within ``allowed`` and the rounding to its type, past which numbers are infinite."""
    t = got.dtype
    bar = allowed * (1 + half_step(t)) + want.abs() * half_step(t) + tiny(t)
    got = got.cpu().double()
    past = got.isinf() & (got.sign() == want.sign()) & (want.abs() + bar >= torch.finfo(t).max * (1 + half_step(t) / 2))
    err = (got - want).abs()
    assert ((err <= bar) | past).all(), ((err / bar).max(), (~((err <= bar) | past)).nonzero()[:5])


def attention_case(pkg, dev, t, b, heads, group, d, lq, lengths, starts, width, seed=0, scale=None, spread=9, long=None):
    scale = d ** -0.5 if scale is None else scale
    cache, ref, table = filled(pkg, dev, b, heads, d, width, seed, lengths, spread)
    q = rand((b, heads * group, lq, d), seed + 7, t)
    got = pkg.ops.cache4_attention(q.to(dev), cache, longer(table, long).to(dev), lengths.to(dev), scale,
                                   starts=None if starts is None else starts.to(dev))
    assert got.dtype == t and got.shape == q.shape
    want, allowed = attention_reference(ref, q, table, lengths, scale, starts, long is not None)
    agree(got, want, allowed)


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize(("heads", "group", "lq"), [(1, 1, 1), (2, 4, 1), (3, 1, 5), (1, 8, 3), (2, 2, 40), (1, 3, 150), (1, 40, 1)])
def test_attention_matches_float64(pkg, dev, heads, group, lq, d, t) -> None:
    """Lengths of none, one, page ends and their neighbours; NaN behind every length."""
    lengths = ints(0, 1, 63, 64, 65, 300, 448)
    attention_case(pkg, dev, t, 7, heads, group, d, lq, lengths, None, 7, seed=d + lq)


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize(("heads", "group", "lq"), [(2, 4, 1), (1, 2, 7), (2, 1, 64), (1, 3, 131), (2, 4, 200)])
def test_attention_causal(pkg, dev, heads, group, lq, d, t) -> None:
    """Queries behind held tokens (none, some), with rows that see nothing (a start before 0) and a
    length below the last query's position."""
    starts = ints(0, 1, 100, -3, 250, 63)
    lengths = ints(lq, lq + 1, 100 + lq, lq, 250 + max(lq // 2, 1), 63 + lq)
    attention_case(pkg, dev, t, 6, heads, group, d, lq, lengths, starts, 8, seed=d + lq)


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize(("heads", "group", "lq"), [(1, 1, 128), (2, 1, 129), (1, 3, 50), (2, 4, 65), (1, 130, 1)])
def test_attention_of_many_rows(pkg, dev, heads, group, lq, d, t) -> None:
    """128 rows of a cache head and more: the last tile with one row, or full; lengths and starts as above; values whose
    scales fp16 holds in all pages, and in some."""
    starts = ints(0, 1, 100, -3, 250, 63)
    lengths = ints(lq, lq + 1, 100 + lq, lq, 250 + max(lq // 2, 1), 63 + lq)
    for spread in (5, 30):
        attention_case(pkg, dev, t, 7, heads, group, d, lq, ints(0, 1, 63, 64, 65, 300, 448), None, 7, seed=d + lq, long=LONG, spread=spread)
        attention_case(pkg, dev, t, 6, heads, group, d, lq, lengths, starts, 8, seed=d + lq, long=LONG, spread=spread)


@gpu
@pytest.mark.parametrize("d", DIMS)
def test_attention_of_many_rows_in_parts(pkg, dev, d) -> None:
    """Sequences of unequal lengths spread over several workgroups, some of which find nothing to do."""
    attention_case(pkg, dev, torch.float16, 3, 1, 2, d, 70, ints(5000, 700, 1), None, 80, long=LONG)
    attention_case(pkg, dev, torch.bfloat16, 3, 1, 1, d, 200, ints(5000, 700, 200), ints(4800, 500, 0), 80, long=LONG)


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
def test_attention_of_pages_beyond_fp16(pkg, dev, d, t) -> None:
    """Single blocks whose scales fp16 does not hold, of keys or values, in the first, a middle or the last page: shared
    pages go another way from there on."""
    for slot, which in ((0, "k"), (1, "v"), (3, "k"), (4, "v"), (6, "v"), (6, "k")):
        cache, _, table = filled(pkg, dev, 1, 1, d, 7, seed=slot, spread=3)
        scales = (cache.k_scales if which == "k" else cache.v_scales).view(torch.uint8)
        scales[int(table[0, slot]), 0, d // 32 - 1, 17 * slot % 50] = 60 if which == "k" else 150
        ref, q = Pages(cache), rand((1, 2, 130, d), 7, t)
        got = pkg.ops.cache4_attention(q.to(dev), cache, longer(table, LONG).to(dev), ints(440).to(dev), d ** -0.5, starts=ints(310).to(dev))
        want, allowed = attention_reference(ref, q, table, ints(440), d ** -0.5, ints(310), True)
        agree(got, want, allowed)


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
def test_attention_does_not_feel_what_stands_behind_a_sequence(pkg, dev, d, t) -> None:
    """Any codes and any scales behind the length and in the table's other pages: the same bits."""
    cache, _, table = filled(pkg, dev, 2, 1, d, 7, seed=1, spread=3)
    lengths = ints(300, 64)
    for lq, long in ((1, None), (150, None), (150, LONG)):
        q = rand((2, 2, lq, d), 7, t).to(dev)
        for starts in (None, (lengths - lq).to(dev)):
            results = []
            for seed in range(3):
                g = torch.Generator().manual_seed(seed)
                for i, n in enumerate(lengths.tolist()):
                    for slot in range(n // 64, 7):
                        page, lo = int(table[i, slot]), max(n - 64 * slot, 0)
                        for x in (cache.k, cache.v):
                            x[page, :, lo:] = torch.randint(0, 256, x[page, :, lo:].shape, dtype=torch.uint8, generator=g).to(dev)
                        for x in (cache.k_scales, cache.v_scales):
                            x = x.view(torch.uint8)[page, :, :, lo:]
                            x.copy_(torch.randint(0, 256, x.shape, dtype=torch.uint8, generator=g))
                results.append(pkg.ops.cache4_attention(q, cache, longer(table, long).to(dev), lengths.to(dev), 0.1, starts=starts))
            assert results[0].isfinite().all()
            assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


@gpu
@pytest.mark.parametrize(("b", "heads", "group", "d", "n"), [(2, 1, 2, 32, 9000), (1, 1, 1, 64, 20000), (2, 2, 8, 128, 9001), (1, 1, 4, 256, 5000)])
def test_attention_long(pkg, dev, b, heads, group, d, n) -> None:
    lengths = ints(*[n - 77 * i for i in range(b)])
    attention_case(pkg, dev, torch.float16, b, heads, group, d, 1, lengths, None, -(-n // 64) + 1)
    attention_case(pkg, dev, torch.bfloat16, b, heads, group, d, 3, lengths, lengths - 3, -(-n // 64) + 1)


@gpu
def test_cache_beyond_4_gib(pkg, dev) -> None:
    """Pages whose offsets pass 32 bits, written and read like the first ones."""
    heads, d, far, width = 4, 128, 280000, 20
    small, big = pkg.ops.Cache4.empty(width, heads, d, dev), pkg.ops.Cache4.empty(far, heads, d, dev)
    low = torch.arange(width, dtype=torch.int32, device=dev)[None]
    high = far - 1 - 7 * low
    k, v = rand((1, heads, 1200, d), 1).to(dev), rand((1, heads, 1200, d), 2).to(dev)
    for cache, table in ((small, low), (big, high)):
        pkg.ops.cache4_append(cache, k, v, table, ints(3).to(dev))
    n = ints(1203).to(dev)
    for mine, theirs in zip(pkg.ops.cache4_read(small, low, n, 1203), pkg.ops.cache4_read(big, high, n, 1203)):
        assert torch.equal(mine, theirs)
    for lq, long in ((1, None), (150, LONG)):
        q = rand((1, 8, lq, d), 3, torch.bfloat16).to(dev)
        got = pkg.ops.cache4_attention(q, big, longer(high, long), n, 0.1)
        assert torch.equal(got, pkg.ops.cache4_attention(q, small, longer(low, long), n, 0.1))


@gpu
@pytest.mark.parametrize("lq", [1, 3, 200])
@pytest.mark.parametrize("d", DIMS)
def test_attention_in_place(pkg, dev, d, lq) -> None:
    cache, _, table = filled(pkg, dev, 2, 2, d, 60)
    q = rand((2, lq, 4, d), 3, torch.bfloat16).to(dev).transpose(1, 2)
    args = cache, longer(table, LONG if lq > 100 else None).to(dev), ints(3800, 640).to(dev), 0.1
    want = pkg.ops.cache4_attention(q, *args)
    got = pkg.ops.cache4_attention(q, *args, out=q)
    assert got is q and torch.equal(got, want)


@gpu
@pytest.mark.parametrize("lq", [2, 140])
@pytest.mark.parametrize("d", DIMS)
def test_attention_value_scales_far_apart(pkg, dev, d, lq) -> None:
    """Values up to 2^80 apart, in both orders."""
    long = LONG if lq > 100 and d > 32 else None
    attention_case(pkg, dev, torch.bfloat16, 2, 1, 1, d, lq, ints(1000, 640), None, 16, spread=40, long=long)
    attention_case(pkg, dev, torch.bfloat16, 2, 1, 1, d, lq, ints(1000, 640), ints(1000 - lq, 500), 16, seed=5, spread=40, long=long)


@gpu
@pytest.mark.parametrize("lq", [1, 4, 100])
def test_attention_scores_far_apart(pkg, dev, lq) -> None:
    """Large scores: one key takes all, probabilities underflow, the running maximum rises often."""
    attention_case(pkg, dev, torch.float16, 2, 2, 2, 64, lq, ints(300, 129), None, 5, scale=3.0)
    attention_case(pkg, dev, torch.bfloat16, 2, 2, 2, 128, lq, ints(300, 129), ints(200, 100), 5, scale=-2.0)
    attention_case(pkg, dev, torch.float16, 2, 1, 2, 64, lq, ints(300, 129), None, 5, scale=0.0)
    if lq == 100:
        attention_case(pkg, dev, torch.float16, 2, 2, 2, 64, lq, ints(300, 129), None, 5, scale=3.0, long=LONG)
        attention_case(pkg, dev, torch.bfloat16, 2, 2, 2, 128, lq, ints(300, 129), ints(200, 100), 5, scale=-2.0, long=LONG)
        attention_case(pkg, dev, torch.float16, 2, 1, 2, 64, lq, ints(300, 129), None, 5, scale=0.0, long=LONG)


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize(("lq", "d"), [(1, 32), (3, 64), (20, 128), (2, 256), (130, 64), (130, 128), (130, 256)])
def test_attention_of_huge_scores(pkg, dev, lq, d, t) -> None:
    """Scores of 2^20 to 2^37, whose last place is up to 2^14: the key of the largest takes all."""
    n = 500
    cache = pkg.ops.Cache4.empty(10, 2, d, dev)
    table = tables(1, 8)
    k, v = rand((1, 2, n, d), 1, scale=100.0), rand((1, 2, n, d), 2)
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), ints(0).to(dev))
    kk, vv = Pages(cache).read(table[0], n)
    best = torch.randint(0, n, (lq,), generator=torch.Generator().manual_seed(3))
    q = torch.stack([kk[h, best] * 100 for h in range(2)])[None].to(t)    # towards one key each
    for scale in (2.0 ** -4, 1.0, 37.3, 1000.0):
        s = q[0].double() @ kk.transpose(1, 2) * scale
        off = (2 * d + 6) * 2.0 ** -24 * (q[0].double().abs() @ kk.abs().transpose(1, 2) * scale).amax(-1)
        top = s.topk(2, -1)
        sure = top.values[..., 0] - top.values[..., 1] > 2 * off + 40      # ahead by more than fp32 scores are off
        assert sure.double().mean() > 0.9
        want = torch.stack([vv[h, top.indices[h, :, 0]] for h in range(2)])
        got = pkg.ops.cache4_attention(q.to(dev), cache, longer(table, LONG if lq > 100 else None).to(dev), ints(n).to(dev), scale).cpu().double()
        bad = (got[0] - want).abs() > want.abs() * (half_step(t) + 2.0 ** -10) + tiny(t)
        assert not (bad & sure[..., None]).any(), scale


@gpu
@pytest.mark.parametrize("x", [15.3, 18.7, 20.5, 22.5, 23.6, 25.2])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize(("b", "n", "lq", "d"), [(1, 100_000, 1, 64), (300, 8_000, 2, 128), (600, 8_000, 1, 32), (600, 4_000, 1, 256),
                                                 (1, 30_000, 130, 64), (1, 30_000, 130, 128), (1, 30_000, 130, 256)])
def test_attention_keeps_the_weight_of_a_long_tail(pkg, dev, b, n, lq, d, first, x) -> None:
    """One key, the first or the last, that outweighs each of ``n`` others by 2^x; their values are 1, its own 0
    in half of the channels and -1 in the others."""
    width, at = -(-(n + 1) // 64), 0 if first else n
    cache = pkg.ops.Cache4.empty(width, 1, d, dev)
    k, v = torch.zeros(1, 1, n + 1, d), torch.ones(1, 1, n + 1, d)
    k[0, 0, at], v[0, 0, at, :d // 2], v[0, 0, at, d // 2:] = 16.0, 0.0, -1.0
    table = torch.arange(width, dtype=torch.int32)[None]
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), ints(0).to(dev))
    p = 2.0 ** -x
    l = 1 + n * p
    o = torch.tensor([n * p / l, (n * p - 1) / l]).double().repeat_interleave(d // 2)
    mass = torch.tensor([n * p / l, (n * p + 1) / l]).double().repeat_interleave(d // 2)
    # Probabilities are taken with 11 bits at least, 2^-32 of the largest at worst; exponents of at most 28 are off by
    # 2^-23 of their size and the exponential by 2^-22: 2^-18 in all. fp32 sums of at most 2,200 additions in a row (a
    # product's sixteens, pages, waves and parts).
    off = n * (p * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -32) * (1 - o) / l * (1 + 2.0 ** -10)
    allowed = off + 2200 * 2.0 ** -24 * (mass + o.abs())
    for t in HALF:
        q = torch.ones(b, 1, lq, d, dtype=t, device=dev)
        got = pkg.ops.cache4_attention(q, cache, longer(table, LONG if lq > 100 else None).expand(b, -1).contiguous().to(dev),
                                       torch.full((b,), n + 1, dtype=torch.int32, device=dev), x * math.log(2.0) / (16 * d))
        err = (got.cpu().double() - o).abs()
        bar = allowed * (1 + half_step(t)) + o.abs() * half_step(t) + tiny(t)
        assert (err <= bar).all(), (err / bar).amax((0, 1, 2))


@gpu
@pytest.mark.parametrize("byte", [0, 1, 2, 20, 90, 100])
@pytest.mark.parametrize(("lq", "d"), [(1, 32), (2, 64), (3, 128), (1, 256), (150, 64), (130, 128), (130, 256)])
def test_attention_of_small_scales(pkg, dev, lq, d, byte) -> None:
    """Keys down to 2^-128 beside large queries, whose scores are ordinary, and values as small."""
    cache, _, table = filled(pkg, dev, 1, 1, d, 3)
    g = torch.Generator().manual_seed(1)
    cache.k_scales.view(torch.uint8).fill_(byte)
    cache.v_scales.view(torch.uint8).fill_(byte)
    big = min(125 - byte, 117)
    q = ((torch.randint(0, 2, (1, 1, lq, d), generator=g) * 2.0 - 1) * 2.0 ** big).to(torch.bfloat16)
    ref = Pages(cache)
    for scale in (2.0 ** -8, 0.4, 3.0):
        got = pkg.ops.cache4_attention(q.to(dev), cache, longer(table, LONG if lq > 100 else None).to(dev), ints(190).to(dev), scale).cpu().double()
        want, allowed = attention_reference(ref, q, table, ints(190), scale, None, lq > 100)
        bar = allowed * (1 + half_step(q.dtype)) + want.abs() * half_step(q.dtype) + tiny(q.dtype) + 2.0 ** -126
        assert ((got - want).abs() <= bar).all(), (scale, ((got - want).abs() / bar).max())


@gpu
@pytest.mark.parametrize(("lq", "d"), [(1, 64), (9, 64), (70, 128), (200, 64), (130, 128), (130, 256), (20, 32)])
def test_attention_loud_tokens_of_small_weight(pkg, dev, lq, d) -> None:
    """Tokens whose values are 2^30 times the others' but whose keys nobody attends to, in one block of channels: the small
    values of the others come out as they are, beside them and in other blocks."""
    cache, _, table = filled(pkg, dev, 1, 1, d, 4, seed=3)
    q = torch.ones(1, 1, lq, d, dtype=torch.float16, device=dev)
    k, v = torch.zeros(1, 1, 256, d, device=dev), rand((1, 1, 256, d), 4).to(dev)
    k[:, :, 64:128] = -16.0
    v[:, :, 64:128, :32] *= 2.0 ** 30
    pkg.ops.cache4_append(cache, k, v, table.to(dev), ints(0).to(dev))
    got = pkg.ops.cache4_attention(q, cache, longer(table, LONG if lq > 100 else None).to(dev), ints(256).to(dev), 1.0).cpu().double()
    want, _ = attention_reference(Pages(cache), q.cpu(), table, ints(256), 1.0, None)
    # equal probabilities of 1: their rounding is exact, the sums are fp32
    assert ((got - want).abs() <= want.abs() * half_step(torch.float16) + 300 * 2.0 ** -23 * 4).all()


@gpu
@pytest.mark.parametrize(("lq", "group", "d", "long"), [
    (4, 1, 64, None), (70, 1, 64, None), (33, 4, 128, None), (200, 1, 32, None), (100, 2, 256, None), (200, 1, 64, LONG),
    (130, 2, 128, LONG), (300, 1, 256, LONG)])
@pytest.mark.parametrize("byte", [255, 254, 253])
def test_attention_nan_in_tokens_that_a_query_does_not_see(pkg, dev, lq, group, d, long, byte) -> None:
    """A NaN key and a NaN value: queries before them are untouched, queries from them on are NaN (in that block of channels,
    for a value); scales whose values pass fp32 touch no query that does not see them either. Where pages are shared the
    others' probabilities are rounded to 16 bits instead of to fp16, as everywhere beside such scales."""
    cache, _, table = filled(pkg, dev, 1, 1, d, 7, seed=1, spread=3)
    q = rand((1, group, lq, d), 2, torch.float16)
    args = (longer(table, long).to(dev), ints(100 + lq).to(dev), d ** -0.5)
    starts = ints(100)
    run = lambda: pkg.ops.cache4_attention(q.to(dev), cache, *args, starts=starts.to(dev)).cpu()
    clean = run()
    want, allowed = attention_reference(Pages(cache), q, table, ints(100 + lq), d ** -0.5, starts, long is not None)
    bar = allowed * (1 + half_step(q.dtype)) + want.abs() * half_step(q.dtype) + tiny(q.dtype)

    def untouched(got, *where):
        if long is None:
            assert torch.equal(got[where], clean[where])
        assert ((got.double() - want).abs() <= bar)[where].all()

    at, blk = 100 + lq // 2, d // 32 - 1
    page, slot = int(table[0, at // 64]), at % 64
    mine = list(range(32 * blk, 32 * blk + 32))
    rest = [i for i in range(d) if i not in mine]
    scales = cache.v_scales.view(torch.uint8)
    was = scales[page, 0, blk, slot].clone()
    scales[page, 0, blk, slot] = byte
    got = run()
    untouched(got, slice(None), slice(None), slice(0, lq // 2))
    untouched(got, Ellipsis, rest)
    if byte == 255:
        assert got[:, :, lq // 2:, mine].isnan().all()
    scales[page, 0, blk, slot] = was
    cache.k_scales.view(torch.uint8)[page, 0, blk, slot] = byte
    got = run()
    untouched(got, slice(None), slice(None), slice(0, lq // 2))
    if byte == 255:
        assert got[:, :, lq // 2:].isnan().all()


@gpu
@pytest.mark.parametrize(("lq", "long"), [(1, None), (90, None), (150, None), (150, LONG)])
def test_attention_says_when_a_page_or_a_length_is_wrong(pkg, dev, lq, long) -> None:
    cache, _, table = filled(pkg, dev, 4, 2, 64, 5, seed=1)
    q = rand((4, 2, lq, 64), 2, torch.float16).to(dev)
    lengths = ints(320, 320, 130, 320)
    good = pkg.ops.cache4_attention(q, cache, longer(table, long).to(dev), lengths.to(dev), 0.1)
    table[1, 3], table[2, 3], table[3, 1] = 1 << 30, -7, -1      # sequence 2 does not reach its bad page
    got = pkg.ops.cache4_attention(q, cache, longer(table, long).to(dev), lengths.to(dev), 0.1)
    assert torch.equal(got[[0, 2]], good[[0, 2]]) and got[[1, 3]].isnan().all()
    got = pkg.ops.cache4_attention(q, cache, longer(table, long).to(dev), ints(320, -4, (long or 5) * 64 + 1, 1 << 30).to(dev), 0.1)
    assert torch.equal(got[0], good[0]) and (got[1] == 0).all() and got[2:].isnan().all()


@gpu
@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize(("lq", "width"), [(1, 9), (70, 9), (140, LONG), (1, 300)])
def test_attention_layouts(pkg, dev, lq, width, d) -> None:
    """Head-interleaved q and out, a table that is part of a wider one, out given."""
    cache, _, table = filled(pkg, dev, 2, 2, d, 5, seed=1)
    q = rand((2, 4, lq, d), 2, torch.bfloat16).to(dev)
    lengths = ints(300, 90).to(dev)
    wide = torch.full((2, width), -1, dtype=torch.int32)
    wide[:, 2:7] = table
    want = pkg.ops.cache4_attention(q, cache, wide.to(dev)[:, 2:width - 2].contiguous(), lengths, 0.1)
    inter = q.transpose(1, 2).contiguous().transpose(1, 2)
    buf = torch.zeros(2, lq, 4, d + 3, dtype=torch.bfloat16, device=dev)
    out = buf[..., 1:d + 1].transpose(1, 2)
    got = pkg.ops.cache4_attention(inter, cache, wide.to(dev)[:, 2:width - 2], lengths, 0.1, out=out)
    assert got is out and torch.equal(out, want)
    assert (buf[..., 0] == 0).all() and (buf[..., d + 1:] == 0).all()


@gpu
def test_cache_refuses_on_the_device(pkg, dev) -> None:
    ops = pkg.ops
    cache = ops.Cache4.empty(4, 2, 64, dev)
    q = torch.zeros(1, 2, 3, 64, dtype=torch.float16, device=dev)
    table, n = torch.zeros(1, 2, dtype=torch.int32, device=dev), ints(5).to(dev)
    ks, vs = cache.k_scales, cache.v_scales
    bad = [ops.Cache4(cache.k, cache.v[:, :1], ks, vs), ops.Cache4(cache.k, cache.v, ks, vs[:, :, :1]), ops.Cache4(cache.k.float(), cache.v, ks, vs),
           ops.Cache4(cache.k, cache.v, ks.view(torch.uint8), vs), ops.Cache4(cache.k[:0], cache.v[:0], ks[:0], vs[:0]),
           ops.Cache4(cache.k.transpose(0, 1).contiguous().transpose(0, 1), cache.v, ks, vs), ops.Cache4(cache.k, cache.v.cpu(), ks, vs),
           ops.Cache4(cache.k[:, :0], cache.v[:, :0], ks[:, :0], vs[:, :0])]
    other = q.clone()
    for call in (*[lambda c=c: ops.cache4_attention(q, c, table, n, 1.0) for c in bad],
                 *[lambda c=c: ops.cache4_read(c, table, n, 5) for c in bad],
                 lambda: ops.cache4_attention(q.float(), cache, table, n, 1.0),
                 lambda: ops.cache4_attention(q[:, :1], cache, table, n, 1.0),
                 lambda: ops.cache4_attention(q[..., :32], cache, table, n, 1.0),
                 lambda: ops.cache4_attention(q, cache, table.long(), n, 1.0),
                 lambda: ops.cache4_attention(q, cache, table[:, :0], n, 1.0),
                 lambda: ops.cache4_attention(q, cache, table, n.repeat(2), 1.0),
                 lambda: ops.cache4_attention(q, cache, table, n, NAN),
                 lambda: ops.cache4_attention(q, cache, table, n, 1.0, out=q[:, :, :2]),
                 lambda: ops.cache4_attention(q, cache, table, n, 1.0, out=q[:, :, :1].expand(-1, -1, 3, -1)),
                 lambda: ops.cache4_attention(q, cache, table, n, 1.0, out=q.view(1, 3, 2, 64).transpose(1, 2)),
                 lambda: ops.cache4_attention(q, cache, table, n, 1.0, starts=n.cpu()),
                 lambda: ops.cache4_append(cache, q, q[:, :, :1], table, n),
                 lambda: ops.cache4_append(cache, q, q.float(), table, n),
                 lambda: ops.cache4_append(cache, q[:, :1], q[:, :1], table, n),
                 lambda: ops.cache4_append(cache, q, q, table, n, counts=n.long()),
                 lambda: ops.cache4_read(cache, table, n, 0), lambda: ops.cache4_read(cache, table, n, 2.0),
                 lambda: ops.cache4_read(cache, table, n, 3, dtype=torch.int8), lambda: ops.cache4_read(cache, table, n[:0], 3),
                 lambda: ops.cache4_read(cache, table, n.long(), 3), lambda: ops.cache4_read(cache, table.repeat(2, 1), n, 3),
                 lambda: ops.cache4_read(cache, table, n, 3, out=(q, q)), lambda: ops.cache4_read(cache, table, n, 2, out=(q, other)),
                 lambda: ops.cache4_read(cache, table, n, 3, out=(q, other.float())),
                 lambda: ops.cache4_read(cache, table, n, 3, out=(q, other[:, :, :1].expand(-1, -1, 3, -1)))):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ together

class Layer:
    """An attention layer on these operators: norm, projection, heads' norm and rotation, append, attention, output
    projection on the residual."""

    def __init__(self, ops, dev, c, heads, kv, d, axes, seed=0):
        self.ops, self.heads, self.kv, self.d = ops, heads, kv, d
        w = lambda o, i, s: ops.quantize8((rand((o, i), seed + s) / math.sqrt(i)).to(dev))
        self.qkv, self.o = w((heads + 2 * kv) * d, c, 1), w(c, heads * d, 2)
        self.g, self.qg, self.kg = ((1 + rand((n,), seed + s, scale=0.1)).to(dev) for n, s in ((c, 5), (d, 6), (d, 7)))
        self.rotary = ops.Rotary.make(axes, device=dev)

    def heads_of(self, x, positions):
        ops = self.ops
        qkv = ops.dense8(ops.rms_norm(x, self.g, quantize=True), self.qkv)
        q, k, v = qkv.unflatten(-1, (-1, self.d)).transpose(1, 2).split([self.heads, self.kv, self.kv], 1)
        q, k = ops.rotate_heads(q, k, positions, self.rotary, q_gamma=self.qg, k_gamma=self.kg)
        return q, k, v

    def __call__(self, x, cache, table, positions, starts, lengths):
        ops, (b, n, c) = self.ops, x.shape
        q, k, v = self.heads_of(x, positions)
        ops.cache4_append(cache, k, v, table, starts)
        a = torch.empty(b, n, self.heads, self.d, dtype=x.dtype, device=x.device)
        ops.cache4_attention(q, cache, table, lengths, self.d ** -0.5, starts=starts, out=a.transpose(1, 2))
        return ops.dense8(ops.quantize8(a.flatten(2)), self.o, residual=x)


def grid_positions(b, grid, dev):
    at = torch.stack(torch.meshgrid(*[torch.arange(n, dtype=torch.int32) for n in grid], indexing="ij")).flatten(1)
    return at[:, None].expand(-1, b, -1).to(dev)


@gpu
def test_layer_prompt_then_tokens(pkg, dev) -> None:
    """A volume's voxels, then tokens one by one: queries, cache and attention against float64 at every step; the whole
    chain repeats bit for bit."""
    b, c, heads, kv, d, grid = 2, 192, 6, 2, 32, (5, 4, 4)
    layer = Layer(pkg.ops, dev, c, heads, kv, d, (8, 12, 12))
    n = math.prod(grid) - 6
    x, at = rand((b, n + 6, c), 9, torch.float16).to(dev), grid_positions(b, grid, dev)

    def go(check=False):
        cache, table = pkg.ops.Cache4.empty(2 * b + 1, kv, d, dev), tables(b, 2, spare=1)
        ref, outs, done = Pages(cache), [], 0
        for step in [n] + [1] * 6:
            starts = torch.full((b,), done, dtype=torch.int32, device=dev)
            part, places = x[:, done:done + step], at[:, :, done:done + step]
            outs.append(layer(part, cache, table.to(dev), places, starts, starts + step))
            if check:
                q, k, v = layer.heads_of(part, places)
                ref.append(k.cpu(), v.cpu(), table, starts.cpu())
                ref.equals(cache)
                want, _ = attention_reference(ref, q.cpu(), table, (starts + step).cpu(), d ** -0.5, starts.cpu())
                got = pkg.ops.cache4_attention(q, cache, table.to(dev), starts + step, d ** -0.5, starts=starts).cpu().double()
                assert (got - want).norm() <= 2.0 ** -11 * want.norm()
            done += step
        return torch.cat(outs, 1), cache

    y, cache = go(True)
    y2, cache2 = go()
    assert torch.equal(y, y2) and torch.equal(cache.k, cache2.k) and torch.equal(cache.v, cache2.v)
    assert y.isfinite().all()


@gpu
def test_captured_step_replays_with_new_inputs(pkg, dev) -> None:
    """One step captured: positions, lengths and tokens come from device memory, so each replay rotates, appends, attends
    and reads at the next position, equal to the eager chain, with eager work between the replays."""
    b, c, heads, kv, d = 3, 128, 4, 2, 64
    layer = Layer(pkg.ops, dev, c, heads, kv, d, (64,), seed=3)
    table = tables(b, 60).to(dev)                       # wide enough for several workgroups a sequence
    x = rand((b, 140, c), 4, torch.float16).to(dev)
    caches = [pkg.ops.Cache4.empty(b * 60 + 2, kv, d, dev) for _ in range(2)]
    starts = torch.zeros(b, dtype=torch.int32, device=dev)
    for cache in caches:
        layer(x[:, :130], cache, table, torch.arange(130, dtype=torch.int32, device=dev)[None].expand(b, -1), starts, starts + 130)
    token, pos = x[:, 130:131].clone(), torch.full((b,), 130, dtype=torch.int32, device=dev)
    ends = pos + 1

    def step(cache, token, pos, ends):
        y = layer(token, cache, table, pos[:, None], pos, ends)
        return y, pkg.ops.cache4_read(cache, table, ends, 2, starts=pos)[0]

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(caches[1], token, pos, ends)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, held = step(caches[1], token, pos, ends)
    for i in range(4):
        token.copy_(x[:, 130 + i:131 + i])
        pos.fill_(130 + i)
        ends.fill_(131 + i)
        graph.replay()
        torch.cuda.synchronize()
        now = torch.full((b,), 130 + i, dtype=torch.int32, device=dev)
        want = step(caches[0], x[:, 130 + i:131 + i], now, now + 1)
        assert torch.equal(y, want[0]) and torch.equal(held, want[1]), i
        assert torch.equal(caches[0].v, caches[1].v) and torch.equal(caches[0].k, caches[1].k)


@gpu
@pytest.mark.parametrize("d", [32, 128])
def test_captured_prompt_replays_at_other_places(pkg, dev, d) -> None:
    """Two graphs of the kernel that shares pages, with and without parts, replayed in turn: queries, starts and lengths
    come from device memory."""
    cache, _, table = filled(pkg, dev, 2, 1, d, 40, seed=2)
    tables2 = [longer(table, LONG).to(dev), longer(table[:1], LONG).to(dev)]
    queries = [rand((b, 2, 150, d), 3 + b, torch.float16).to(dev) for b in (2, 1)]
    starts = [torch.zeros(b, dtype=torch.int32, device=dev) for b in (2, 1)]
    ends = [s + 150 for s in starts]
    run = lambda i: pkg.ops.cache4_attention(queries[i], cache, tables2[i], ends[i], 0.1, starts=starts[i])
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        run(0), run(1)
    torch.cuda.current_stream().wait_stream(warm)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], [None, None]
    for i in range(2):
        with torch.cuda.graph(graphs[i], pool=graphs[0].pool() if i else None):
            outs[i] = run(i)
    for n, at in enumerate((0, 700, 2400, 63, -20)):
        for i in range(2):
            starts[i].fill_(at)
            ends[i].fill_(max(at, 0) + 150 - n)
            queries[i].mul_(-1.5 if n % 2 else 0.75)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], run(i)), (n, i)


@gpu
def test_two_streams_at_once(pkg, dev) -> None:
    """Calls on two streams share nothing: results equal those of one stream."""
    cases = []
    for seed in (1, 2):
        cache, _, table = filled(pkg, dev, 1, 1, 64, 60, seed=seed)
        cases.append((rand((1, 4, 1, 64), seed, torch.float16).to(dev), cache, table.to(dev), ints(3800).to(dev)))
    run = lambda c: (pkg.ops.cache4_attention(*c, 0.1), pkg.ops.cache4_read(*c[1:], 3800)[0])
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
