"""A sequence whose tokens lie in several caches: what each part gives, and what they give together."""
import pytest
import torch

from kv4_reference import check, reference
from test_gpu_kv4 import BF, DEV, HF, _gen, _ints, _table

pytestmark = pytest.mark.gpu


def _parts(sizes, Hkv, D, dt):
    """``sizes[p][b]``: tokens of sequence b in part p.  Caches, tables, and the same tokens in one cache."""
    import opt_ring_flash_attn_b200 as rfa

    B = len(sizes[0])
    total = [sum(s[b] for s in sizes) for b in range(B)]
    k, v = (torch.randn(B, max(total), Hkv, D, generator=_gen(41 + i), device=DEV).to(dt) for i in range(2))

    def fill(lens, begin):
        table, n = _table(lens)
        cache = rfa.KV4Cache.empty(n, Hkv, D, dt, DEV)
        T = max(max(lens), 1)
        at = (torch.tensor(begin, device=DEV)[:, None] + torch.arange(T, device=DEV)).clamp(max=k.shape[1] - 1)
        rows = torch.arange(B, device=DEV)[:, None]
        rfa.kv4_append(cache, k[rows, at], v[rows, at], table, _ints([0] * B), _ints(lens))
        return cache, table

    begin, parts = [0] * B, []
    for s in sizes:
        parts.append(fill(s, begin))
        begin = [a + n for a, n in zip(begin, s)]
    return parts, fill(total, [0] * B), total


SIZES = {
    "two": [[300, 64, 5], [200, 1, 90]],
    "short_last": [[500, 128, 63], [2, 3, 1]],     # fewer tokens than there are queries: the first part holds some of them
    "empty_parts": [[0, 70, 0], [130, 0, 40], [0, 0, 7]],
    "long": [[3000, 10, 1], [1000, 2500, 2]],
}


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("T,Hq,Hkv,D,dt", [(1, 4, 2, 64, BF), (4, 2, 2, 64, HF), (5, 8, 2, 128, BF), (20, 4, 1, 128, HF),
                                           (3, 4, 4, 256, BF), (2, 3, 1, 96, BF), (7, 2, 1, 192, HF)])
@pytest.mark.parametrize("scores", ["plain", "both"])
def test_parts(sizes, T, Hq, Hkv, D, dt, scores):
    import opt_ring_flash_attn_b200 as rfa

    sizes = SIZES[sizes]
    parts, (cache, table), total = _parts(sizes, Hkv, D, dt)
    B = len(total)
    q = torch.randn(B, T, Hq, D, generator=_gen(43), device=DEV).to(dt)
    kw, ref_kw = {}, {}
    if scores == "both":
        slopes = torch.tensor([2.0 ** (-4.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)
        kw, ref_kw = dict(softcap=5.0, alibi_slopes=slopes), dict(softcap=5.0, slopes=slopes)
    left = list(total)
    got, refs = [], []
    for s, (c, t) in zip(sizes, parts):
        left = [a - n for a, n in zip(left, s)]
        got.append(rfa.kv4_attn_with_lse(q, c, t, _ints(s), tokens_after=_ints(left), **kw))
        refs.append(reference(q, c, t, s, after=left, **ref_kw))
        rfa.check("test")
        check(*got[-1], refs[-1])
    whole = reference(q, cache, table, total, **ref_kw)
    lse = torch.stack([x.double() for _, x in got])
    top = torch.logsumexp(lse, 0)
    w = torch.exp(lse - top.masked_fill(top.isinf(), 0)).transpose(2, 3)[..., None]  # [parts, B, T, Hq, 1]
    joined = sum(wp * o.double() for wp, (o, _) in zip(w, got))
    # each part by its weight; a weight is off by twice the largest error of an lse
    off = 2 * torch.stack([r[3] for r in refs]).amax(0).transpose(1, 2)[..., None]
    bound = sum(wp * (r[1] + off * o.double().abs()) for wp, r, (o, _) in zip(w, refs, got)) + 1e-12
    over = ((joined - whole[0]).abs() / bound).max()
    assert over <= 1, f"{over.item():.2f} of the bound"
    assert torch.equal(top.isinf(), whole[2].isinf())
    if len(sizes) == 2 and min(map(min, sizes)) > 0:
        # the last part by itself is a plain call
        a = rfa.kv4_attn_with_lse(q, *parts[-1], _ints(sizes[-1]), **kw)
        assert torch.equal(a[0], got[-1][0]) and torch.equal(a[1], got[-1][1])


def test_offsets_at_the_ends_of_int32():
    """Negative counts are 0; a part so far ahead of the queries that positions end at 2^31 is safe."""
    import opt_ring_flash_attn_b200 as rfa

    parts, _, _ = _parts([[100, 100, 100, 100]], 1, 64, BF)
    q = torch.randn(4, 2, 2, 64, generator=_gen(44), device=DEV).to(BF)
    out, lse = rfa.kv4_attn_with_lse(q, *parts[0], _ints([100] * 4), tokens_after=_ints([-2 ** 31, -1, 0, 2 ** 31 - 1]))
    rfa.check("test")
    check(out, lse, reference(q, *parts[0], [100] * 4, after=[0, 0, 0, 2 ** 31 - 101]))


@pytest.mark.parametrize("D,dt,Hq,Hkv,size", [(128, BF, 8, 2, 130), (64, HF, 4, 4, 64), (256, BF, 4, 1, 100), (96, HF, 6, 2, 257)])
def test_a_prompt_in_parts(D, dt, Hq, Hkv, size):
    """A prompt goes in part by part: each part is appended and attends to all that is cached, a ragged last one too."""
    import opt_ring_flash_attn_b200 as rfa

    B, S = 2, 600
    x = [torch.randn(B, S, h, D, generator=_gen(45 + i), device=DEV).to(dt) for i, h in enumerate((Hq, Hkv, Hkv))]
    slopes = torch.tensor([2.0 ** (-4.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)
    table, n = _table([S] * B)
    cache = rfa.KV4Cache.empty(n, Hkv, D, dt, DEV)
    for a in range(0, S, size):
        e = min(S, a + size)
        rfa.kv4_append(cache, x[1][:, a:e], x[2][:, a:e], table, _ints([a] * B))
        out, lse = rfa.kv4_attn_with_lse(x[0][:, a:e], cache, table, _ints([e] * B), softcap=20.0, alibi_slopes=slopes)
        rfa.check("test")
        check(out, lse, reference(x[0][:, a:e], cache, table, [e] * B, softcap=20.0, slopes=slopes))
