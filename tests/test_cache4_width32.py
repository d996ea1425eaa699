"""``cache4_attention`` at head width 32 where many queries share pages, whose kernel has a division of work of its own (two
waves widen keys, two values): the special values that the other head widths are tested with."""

from __future__ import annotations

import pytest
import torch

from tests import test_ops4 as ops4
from tests.test_ops4 import HALF, LONG, ints

gpu = pytest.mark.gpu


@pytest.mark.parametrize("lq", [130, 150, 200, 300])
def test_these_calls_share_pages(pkg, lq) -> None:
    import ctypes
    lib = pkg._lib
    for group in (1, 2):
        a = lib.Cache4AttentionArgs(cache=ops4._cache_args(lib, heads=1, head_dim=32), batch=1, q_heads=group, q_len=lq, q=16, o=16,
                                    scale=1.0, table=16, table_pitch=LONG, width=LONG, lengths=16)
        assert lib.lib.ldx_cache4_attention_rows(ctypes.byref(a)) == 128


@gpu
@pytest.mark.parametrize("x", [15.3, 18.7, 20.5, 22.5, 23.6, 25.2])
@pytest.mark.parametrize("first", [True, False])
def test_long_tail(pkg, dev, first, x) -> None:
    ops4.test_attention_keeps_the_weight_of_a_long_tail(pkg, dev, 1, 30_000, 130, 32, first, x)


@gpu
@pytest.mark.parametrize("byte", [0, 1, 2, 20, 90, 100])
@pytest.mark.parametrize("lq", [130, 150])
def test_small_scales(pkg, dev, lq, byte) -> None:
    ops4.test_attention_of_small_scales(pkg, dev, lq, 32, byte)


@gpu
@pytest.mark.parametrize("lq", [130, 200])
def test_loud_tokens_of_small_weight(pkg, dev, lq) -> None:
    ops4.test_attention_loud_tokens_of_small_weight(pkg, dev, lq, 32)


@gpu
@pytest.mark.parametrize("byte", [255, 254, 253])
@pytest.mark.parametrize(("lq", "group"), [(200, 1), (130, 2), (300, 1)])
def test_nan_in_tokens_that_a_query_does_not_see(pkg, dev, lq, group, byte) -> None:
    """(All channels are one block here, so that there are no others beside a value of NaN.)"""
    ops4.test_attention_nan_in_tokens_that_a_query_does_not_see(pkg, dev, lq, group, 32, LONG, byte)


@gpu
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("spread", [20, 40])
def test_value_scales_far_apart(pkg, dev, spread, t) -> None:
    ops4.attention_case(pkg, dev, t, 2, 1, 1, 32, 140, ints(1000, 640), None, 16, spread=spread, long=LONG)
    ops4.attention_case(pkg, dev, t, 2, 1, 1, 32, 140, ints(1000, 640), ints(860, 500), 16, seed=5, spread=spread, long=LONG)


@gpu
def test_scores_far_apart(pkg, dev) -> None:
    for t, scale, starts in ((torch.float16, 3.0, None), (torch.bfloat16, -2.0, ints(200, 100)), (torch.float16, 0.0, None)):
        ops4.attention_case(pkg, dev, t, 2, 2, 2, 32, 100, ints(300, 129), starts, 5, scale=scale, long=LONG)


@gpu
def test_says_when_a_page_or_a_length_is_wrong(pkg, dev) -> None:
    cache, _, table = ops4.filled(pkg, dev, 4, 2, 32, 5, seed=1)
    q = ops4.rand((4, 2, 150, 32), 2, torch.float16).to(dev)
    attend = lambda lengths: pkg.ops.cache4_attention(q, cache, ops4.longer(table, LONG).to(dev), ints(*lengths).to(dev), 0.1)
    good = attend((320, 320, 130, 320))
    table[1, 3], table[2, 3], table[3, 1] = 1 << 30, -7, -1      # sequence 2 does not reach its bad page
    got = attend((320, 320, 130, 320))
    assert torch.equal(got[[0, 2]], good[[0, 2]]) and got[[1, 3]].isnan().all()
    got = attend((320, -4, LONG * 64 + 1, 1 << 30))
    assert torch.equal(got[0], good[0]) and (got[1] == 0).all() and got[2:].isnan().all()
