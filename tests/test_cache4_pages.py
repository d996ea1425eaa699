"""``cache4_attention`` where many queries share pages that fp16 does not hold, with and without NaN among their values."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_ops4 import DIMS, HALF, LONG, Pages, attention_reference, filled, half_step, ints, longer, rand, tiny

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize(("slot", "token", "block"), [(None, 0, 0), (0, 0, 0), (2, 63, -1), (3, 5, 0), (4, 40, -1), (4, 63, 0)])
def test_values_beyond_fp16_in_every_page(pkg, dev, slot, token, block, d, t) -> None:
    """A block of values too small for fp16 in every page, and a NaN in the first or last token or block of one: queries that
    see it have NaN in that block, all else is as without."""
    n, lq = 310, 130
    cache, _, table = filled(pkg, dev, 1, 1, d, 5, seed=d, spread=3)
    scales = cache.v_scales.view(torch.uint8)
    for s in range(5):
        scales[int(table[0, s]), 0, s % (d // 32), 7 + s] = 60
    q, starts = rand((1, 2, lq, d), 7, t), ints(n - lq)
    want, allowed = attention_reference(Pages(cache), q, table, ints(n), d ** -0.5, starts, True)
    if slot is not None:
        at, block = 64 * slot + token, block % (d // 32)
        scales[int(table[0, slot]), 0, block, token] = 255
        if at < n:
            want[:, :, max(at - (n - lq), 0):, 32 * block:32 * block + 32] = math.nan
    got = pkg.ops.cache4_attention(q.to(dev), cache, longer(table, LONG).to(dev), ints(n).to(dev), d ** -0.5, starts=starts.to(dev))
    got = got.cpu().double()
    bar = allowed * (1 + half_step(t)) + want.abs() * half_step(t) + tiny(t)
    assert torch.equal(got.isnan(), want.isnan())
    assert (((got - want).abs() <= bar) | want.isnan()).all()
