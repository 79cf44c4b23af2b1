"""The 4-bit cache's attention against bounds that follow each group of 32 channels (kv4_reference): ordinary values at every
shape, then scales of V that lie far apart between the groups of one token."""
import math

import pytest
import torch

from kv4_reference import check, reference
from test_gpu_kv4 import BF, DEV, HF, _filled, _gen, _ints, _table

pytestmark = pytest.mark.gpu

LENS = {"short": [1, 0, 5, 64, 65], "edges": [63, 128, 129, 700], "long": [3001]}


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("D,dt,Hq,Hkv,T", [(64, BF, 2, 2, 1), (128, BF, 8, 1, 1), (128, HF, 8, 2, 4), (96, HF, 3, 1, 5),
                                           (192, BF, 4, 2, 2), (256, HF, 4, 4, 1), (256, BF, 16, 1, 3), (64, HF, 12, 1, 8),
                                           (128, BF, 5, 5, 20), (128, BF, 16, 1, 1), (64, BF, 12, 1, 2)])
@pytest.mark.parametrize("scores", ["plain", "cap", "bias"])
def test_every_shape(lens, D, dt, Hq, Hkv, T, scores):
    import opt_ring_flash_attn_b200 as rfa

    lens = LENS[lens]
    cache, table, _ = _filled(21, lens, Hkv, D, dt)
    q = torch.randn(len(lens), T, Hq, D, generator=_gen(25), device=DEV).to(dt)
    kw = {}
    if scores != "plain":
        kw["softcap"] = 3.0
    slopes = None
    if scores == "bias":
        slopes = kw["alibi_slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints(lens), **kw)
    rfa.check("test")
    check(out, lse, reference(q, cache, table, lens, softcap=kw.get("softcap", 0.0), slopes=slopes))


def _one(dt, D, n, v, seed=31):
    import opt_ring_flash_attn_b200 as rfa

    table, pool = _table([n])
    cache = rfa.KV4Cache.empty(pool, 1, D, dt, DEV)
    k = torch.randn(1, n, 1, D, generator=_gen(seed), device=DEV).to(dt)
    rfa.kv4_append(cache, k, v.to(dt), table, _ints([0]))
    return cache, table


@pytest.mark.parametrize("Hq", [4, 8, 16])
@pytest.mark.parametrize("D,dt,ratio", [(128, BF, 2.0 ** 10), (128, BF, 2.0 ** 17), (128, BF, 2.0 ** 40), (64, BF, 2.0 ** 20),
                                        (96, BF, 2.0 ** 20), (192, BF, 2.0 ** 20), (256, BF, 2.0 ** 20), (128, HF, 2.0 ** 13),
                                        (64, HF, 2.0 ** 13), (256, HF, 2.0 ** 13)])
def test_groups_of_a_token_far_apart(D, dt, ratio, Hq):
    """One group of channels holds values ``ratio`` times those of the others: each keeps its own accuracy."""
    import opt_ring_flash_attn_b200 as rfa

    n = 3001
    v = torch.randn(1, n, 1, D, generator=_gen(32), device=DEV)
    v[..., 32:64] *= ratio
    cache, table = _one(dt, D, n, v)
    q = torch.randn(1, 1, Hq, D, generator=_gen(33), device=DEV).to(dt)
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints([n]))
    check(out, lse, reference(q, cache, table, [n]))


@pytest.mark.parametrize("top", [2.0 ** 30, 2.0 ** 100, 2.0 ** 110, 2.0 ** 114])
def test_largest_and_smallest_values(top):
    """V over nearly the whole range of bf16, groups and tokens of either end beside each other (500 weights of 4 at most times
    2^116.2 stay inside fp32)."""
    import opt_ring_flash_attn_b200 as rfa

    n, D = 500, 128
    v = torch.randn(1, n, 1, D, generator=_gen(34), device=DEV)
    v[..., :32] *= top
    v[..., 64:96] /= top
    v[0, 250:, 0, 96:] *= top
    cache, table = _one(BF, D, n, v)
    q = torch.randn(1, 1, 4, D, generator=_gen(35), device=DEV).to(BF)
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints([n]))
    check(out, lse, reference(q, cache, table, [n]))


@pytest.mark.parametrize("dt,size", [(BF, 1e7), (HF, 500.0)])
def test_negative_scales(dt, size):
    """A cache that another program filled: scales below 0, far larger than the others."""
    import opt_ring_flash_attn_b200 as rfa

    n, D = 900, 128
    v = torch.randn(1, n, 1, D, generator=_gen(36), device=DEV)
    cache, table = _one(dt, D, n, v)
    page = table[0, 5].long()
    cache.meta[page, :, 1, :, 2, 0] *= -size
    q = torch.randn(1, 1, 4, D, generator=_gen(37), device=DEV).to(dt)
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints([n]))
    check(out, lse, reference(q, cache, table, [n]))


def test_a_group_that_is_no_number_beside_a_large_one():
    """An infinity keeps to its 32 channels, also where the other groups of its token are the largest so far."""
    import opt_ring_flash_attn_b200 as rfa

    n, D = 900, 128
    v = torch.randn(1, n, 1, D, generator=_gen(38), device=DEV)
    v[0, 400:402] *= 1e7
    v[0, 400:402, 0, 40] = math.inf
    cache, table = _one(BF, D, n, v)
    q = torch.randn(1, 1, 4, D, generator=_gen(39), device=DEV).to(BF)
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints([n]))
    keep = [c for c in range(D) if not 32 <= c < 64]
    assert not torch.isfinite(out[..., 32:64]).any()
    check(out, lse, reference(q, cache, table, [n]), keep)
