"""``cache4_attention`` of scores far beyond what fp32 holds to a whole number, compared with float64. Every check states
what holds (``err <= bar``), which NaN does not."""

from __future__ import annotations

import pytest
import torch

from tests.test_ops4 import (DIMS, HALF, LONG, Pages, agree, attention_reference, filled, half_step, ints, longer, rand, tables,
                             tiny)

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize(("lq", "long"), [(1, None), (40, None), (130, LONG), (300, LONG)])
@pytest.mark.parametrize("down", [False, True])
def test_the_key_of_the_largest_score_takes_all(pkg, dev, lq, long, d, t, down) -> None:
    """Scores of one product each, exact before they are scaled, whose largest are 2^18 to 2^100 (``down``: all of them below
    0) and ahead of the next by a third. Their last place is up to 2^77: whichever way the scaled scores are rounded, the
    largest one's value comes out."""
    n, heads = 500, 2
    cache, table = pkg.ops.Cache4.empty(10, heads, d, dev), tables(1, 8)
    g = torch.Generator().manual_seed(d + lq)
    k, v = torch.zeros(1, heads, n, d), rand((1, heads, n, d), 2)
    k[..., 3] = torch.tensor([-6.0, -4, -3] if down else [-3.0, 1, 2, 3, 4])[torch.randint(0, 3 if down else 5, (1, heads, n), generator=g)]
    best = torch.tensor([(37 * lq + 61 * h) % n for h in range(heads)])
    k[0, torch.arange(heads), best, 3] = -2.0 if down else 6.0
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), ints(0).to(dev))
    values = Pages(cache).read(table[0], n)[1]
    want = values[torch.arange(heads), best][None, :, None]
    # One probability, as it is rounded, over itself: their product is exact where it is fp16, its two parts hold 16 bits where it
    # is not; the division and its product 2^-22.
    bar = want.abs() * (2.0 ** -22 if long else 2.0 ** -16) * (1 + half_step(t)) + want.abs() * half_step(t) + tiny(t)
    q = torch.zeros(1, heads, lq, d)
    q[..., 3] = 1024 * (1 + torch.rand(1, heads, lq, generator=g))
    for sign in (1.0, -1.0):
        for e in (18, 19, 20, 21, 22, 23, 24, 25, 25.5, 26, 26.5, 27, 27.5, 28, 28.5, 29, 30, 31, 33, 36, 50, 100):
            scale = sign * 0.961 * 2.0 ** (e - 13)
            got = pkg.ops.cache4_attention((q * sign).to(t).to(dev), cache, longer(table, long).to(dev), ints(n).to(dev), scale)
            err = (got.cpu().double() - want).abs()
            assert (err <= bar).all(), (sign, e, (~(err <= bar)).sum(), got.isnan().sum())


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize(("lq", "d"), [(1, 32), (3, 64), (20, 128), (2, 256), (130, 32), (130, 64), (130, 128), (130, 256)])
def test_huge_scores_of_all_channels(pkg, dev, lq, d, t) -> None:
    """Queries towards one key each with scores of 2^20 to 2^37: the key of the largest takes all where it is ahead by more
    than fp32 scores are off, and every other result lies among the values."""
    n = 500
    cache, table = pkg.ops.Cache4.empty(10, 2, d, dev), tables(1, 8)
    k, v = rand((1, 2, n, d), 1, scale=100.0), rand((1, 2, n, d), 2)
    pkg.ops.cache4_append(cache, k.to(dev), v.to(dev), table.to(dev), ints(0).to(dev))
    kk, vv = Pages(cache).read(table[0], n)
    best = torch.randint(0, n, (lq,), generator=torch.Generator().manual_seed(3))
    q = torch.stack([kk[h, best] * 100 for h in range(2)])[None].to(t)
    most = vv.abs().amax((1, 2))[:, None, None]
    for scale in (2.0 ** -4, 0.3, 0.71, 1.0, 1.3, 2.9, 37.3, 1000.0):
        s = q[0].double() @ kk.transpose(1, 2) * scale
        off = (2 * d + 6) * 2.0 ** -24 * (q[0].double().abs() @ kk.abs().transpose(1, 2) * scale).amax(-1)
        top = s.topk(2, -1)
        sure = top.values[..., 0] - top.values[..., 1] > 2 * off + 40
        assert sure.double().mean() > 0.9
        want = torch.stack([vv[h, top.indices[h, :, 0]] for h in range(2)])
        got = pkg.ops.cache4_attention(q.to(dev), cache, longer(table, LONG if lq > 100 else None).to(dev), ints(n).to(dev), scale)
        got = got.cpu().double()[0]
        bar = want.abs() * (half_step(t) + 2.0 ** -10) + tiny(t)
        assert (((got - want).abs() <= bar) | ~sure[..., None]).all(), (scale, got.isnan().any(-1).sum())
        assert (got.abs() <= most * (1 + 2 * half_step(t) + 2.0 ** -10)).all(), scale


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize(("lq", "long"), [(40, None), (130, LONG)])
def test_ordinary_queries_beside_those_of_huge_scores(pkg, dev, lq, long, d, t) -> None:
    """Every third query's scores are 2^21 times the others', and the first page's and a middle one's keys are zeros: the ordinary
    queries come out as they do alone, the others take their largest key's value."""
    cache, _, table = filled(pkg, dev, 1, 1, d, 6, seed=d, spread=5)
    zeros, values = torch.zeros(1, 1, 64, d, device=dev), rand((1, 1, 64, d), 5).to(dev)
    for slot in (0, 3):
        pkg.ops.cache4_append(cache, zeros, values, table.to(dev), ints(64 * slot).to(dev))
    ref, n = Pages(cache), 370
    q = rand((1, 2, lq, d), 7, t)
    q[:, :, ::3] *= 2.0 ** 13
    k, v = ref.read(table[0], n)
    ordinary = [i for i in range(lq) if i % 3]
    for scale in (2.0 ** 8, -(2.0 ** 8)):
        x = q.clone()
        x[:, :, ordinary] *= 2.0 ** -8
        got = pkg.ops.cache4_attention(x.to(dev), cache, longer(table, long).to(dev), ints(n).to(dev), scale)
        want, allowed = attention_reference(ref, x, table, ints(n), scale, None, long is not None)
        agree(got[:, :, ordinary], want[:, :, ordinary], allowed[:, :, ordinary])
        s = x[0, :, ::3].double() @ k[0].t().contiguous() * scale
        off = (2 * d + 6) * 2.0 ** -24 * (x[0, :, ::3].double().abs() @ k[0].t().contiguous().abs() * abs(scale)).amax(-1)
        top = s.topk(2, -1)
        sure = top.values[..., 0] - top.values[..., 1] > 2 * off + 40
        assert sure.double().mean() > 0.9
        want = v[0][top.indices[..., 0]]
        bar = want.abs() * (half_step(t) + 2.0 ** -10) + tiny(t)
        err = (got[0, :, ::3].cpu().double() - want).abs()
        assert ((err <= bar) | ~sure[..., None]).all() and got.isfinite().all()
