"""``rotate_heads`` at the ends of its types' ranges, compared with float64: heads of the largest values, gammas
and an eps far from one, and channels that are not turned."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_ops4 import check_rotated, ints, rand

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
WIDE = [torch.bfloat16, torch.float32]   # the types whose values' squares pass fp32


def test_plans_of_odd_arguments(pkg) -> None:
    make = pkg.ops.Rotary.make
    assert torch.equal(make([4, 6], scale=[1.0, 0.5], device="cpu").turns, make((4, 6), scale=(1.0, 0.5), device="cpu").turns)
    for theta in (0.0, -2.0, math.nan):
        with pytest.raises(ValueError, match="theta"):
            make(8, theta=theta, device="cpu")
    with pytest.raises(ValueError, match="scale"):
        make((4, 6), scale=[1.0], device="cpu")


# Heads whose halves, or whose sections' halves, divide by 8, 4, 2 and nothing, of one unit a lane and of several.
PLANS = [((2,), 2), ((32,), 32), ((8, 12, 12), 32), ((36,), 36), ((64,), 64), ((16, 30, 30), 80), ((128,), 128),
         ((256,), 256), ((512,), 512), ((254, 6, 250), 510), ((252, 8, 248), 508)]


@gpu
@pytest.mark.parametrize("t", WIDE)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("axes", "d"), PLANS)
def test_norm_of_heads_of_the_largest_values(pkg, dev, axes, d, interleaved, t) -> None:
    """Every channel the type's largest number of either sign; 2^127, 2^126, 2^64 and 2^60 (squares that pass fp32 only in a
    wide head) times ordinary numbers, held at the type's end; one large channel among ordinary ones."""
    rotary, most = pkg.ops.Rotary.make(axes, interleaved=interleaved), torch.finfo(t).max
    x = rand((1, 7, 3, d), 1).double()
    x[0, 0] = torch.where(x[0, 0] < 0, -most, most)
    for i, e in enumerate((127, 126, 64, 60)):
        x[0, 1 + i] *= 2.0 ** e
    x[0, 5, :, d // 2] = -most
    x = x.clamp(-most, most).to(t)
    at = ints(0, 3, -1000).expand(len(axes), 1, 3)
    gamma = 1 + rand((d,), 3, scale=0.2)
    got = pkg.ops.rotate_heads(x.to(dev), None, at.to(dev), rotary, q_gamma=gamma.to(dev))
    check_rotated(got, x, gamma, 1e-6, at, rotary)


@gpu
@pytest.mark.parametrize("t", WIDE)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("axes", "d"), PLANS)
def test_norm_with_an_eps_beside_large_squares(pkg, dev, axes, d, interleaved, t) -> None:
    """An eps of the size of the mean square, where the squares' sum, or the mean with eps, passes fp32."""
    rotary = pkg.ops.Rotary.make(axes, interleaved=interleaved)
    x = rand((1, 5, 3, d), 1)
    for i, e in enumerate((0, 60, 62.5, 63.5, 66)):
        x[0, i] *= 2.0 ** e
    x, at, gamma = x.to(t), ints(0, 3, -1000).expand(len(axes), 1, 3), 1 + rand((d,), 3, scale=0.2)
    for eps in (1e36, 3e38):
        got = pkg.ops.rotate_heads(x.to(dev), None, at.to(dev), rotary, q_gamma=gamma.to(dev), eps=eps)
        check_rotated(got, x, gamma, torch.tensor(eps, dtype=torch.float32).double(), at, rotary)


@gpu
@pytest.mark.parametrize("t", WIDE)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("axes", "d"), PLANS)
def test_norm_with_gammas_far_from_one(pkg, dev, axes, d, interleaved, t) -> None:
    """Small heads times a large gamma and large ones times a small gamma: the root times gamma leaves fp32, the result does
    not."""
    rotary = pkg.ops.Rotary.make(axes, interleaved=interleaved)
    at = ints(0, 3, -1000).expand(len(axes), 1, 3)
    for size, factor in ((2.0 ** -60, 2.0 ** 90), (2.0 ** 60, 2.0 ** -90), (2.0 ** 120, 2.0 ** -50), (1.0, 2.0 ** 120)):
        x, gamma = (rand((1, 2, 3, d), 1) * size).to(t), (1 + rand((d,), 3, scale=0.2)) * factor
        got = pkg.ops.rotate_heads(x.to(dev), None, at.to(dev), rotary, q_gamma=gamma.to(dev), eps=1e-30)
        check_rotated(got, x, gamma, torch.tensor(1e-30, dtype=torch.float32).double(), at, rotary)


# Sections that leave channels behind them: in both kernels, of a lane's unit as a whole and in its middle.
PARTS = [((8,), 24), ((16, 16), 64), ((32,), 128), ((16, 30, 30), 80), ((10, 6), 18), ((24, 24, 16), 72), ((6,), 36),
         ((2, 2, 2, 2), 14), ((254, 6, 248), 510), ((252, 8, 240), 512), ((2,), 4)]


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("axes", "d"), PARTS)
def test_channels_behind_the_sections_stay(pkg, dev, axes, d, interleaved, t) -> None:
    """NaN, infinities and zeros of both signs in channels that are not turned stay in their own; with a norm an infinity
    makes the other channels zeros, and a NaN all of them NaN."""
    rotary, w = pkg.ops.Rotary.make(axes, interleaved=interleaved), sum(axes)
    q, at = rand((1, 9, 3, d), 1, t), ints(0, 3, -1000).expand(len(axes), 1, 3)
    q[0, 0, :, w], q[0, 1, :, d - 1], q[0, 2, :, (w + d) // 2] = math.inf, -math.inf, math.nan
    q[0, 3, :, w:] = -0.0
    q[0, 4, :, w::2] = -0.0
    q[0, 5, :, w], q[0, 5, :, d - 1] = math.inf, math.nan
    q[0, 6, :, w:] = torch.finfo(t).max
    got = pkg.ops.rotate_heads(q.to(dev), None, at.to(dev), rotary).cpu()
    assert torch.equal(got[..., w:].nan_to_num(7.0, 8.0, 9.0), q[..., w:].nan_to_num(7.0, 8.0, 9.0))
    there = ~q[..., w:].isnan()
    assert torch.equal(got[..., w:].signbit()[there], q[..., w:].signbit()[there])
    finite = torch.where(q.isfinite(), q, 0.0)
    want = pkg.ops.rotate_heads(finite.to(dev), None, at.to(dev), rotary).cpu()
    assert torch.equal(got[..., :w], want[..., :w])
    check_rotated(want, finite, None, 1e-6, at, rotary)

    normed = pkg.ops.rotate_heads(q.to(dev), None, at.to(dev), rotary, q_gamma=torch.ones(d, device=dev)).cpu()
    assert normed[0, [2, 5]].isnan().all()
    for h, c in ((0, w), (1, d - 1)):
        others = [i for i in range(d) if i != c]
        assert normed[0, h, :, c].isnan().all() and (normed[0, h][:, others] == 0).all()
    keep = [3, 4, 7, 8] + [6] * (t == torch.float16)   # (beside other types' largest numbers the turned channels are subnormal)
    check_rotated(normed[:, keep], q[:, keep], torch.ones(d), 1e-6, at, rotary)
    assert torch.equal(normed[0, 3:5, :, w:].signbit(), q[0, 3:5, :, w:].signbit())
