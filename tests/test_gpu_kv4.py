"""The 4-bit K/V cache: codes and values exactly, attention over it against its definition in 64 bits (bounds counted from the
roundings), then the ways it is called."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _table(lens, spare=0, seed=0):
    """Scattered pages for sequences of these lengths, and the size of the pool."""
    counts = [max(1, -(-n // 64)) + spare for n in lens]
    order = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed)).tolist()
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c] + [-1] * (max(counts) - c))
        at += c
    return _ints(rows), sum(counts)


def quantized(x):
    """Values that x reads back as, in 64 bits: the format's definition."""
    g = x.unflatten(-1, (-1, 32)).double()
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    sc = ((hi - lo) / 15).to(x.dtype).double()
    u = torch.where(sc > 0, ((g - lo) / torch.where(sc > 0, sc, 1.0)).round().clamp(0, 15), 0.0)
    return (u * sc + lo).flatten(-2)


def _filled(seed, lens, Hkv, D, dt, std=1.0, spare=0):
    """A cache that holds random tokens, its table, and the values (64 bits) it stands for: [B][len, 2, Hkv, D]."""
    import opt_ring_flash_attn_b200 as rfa

    table, n = _table(lens, spare)
    cache = rfa.KV4Cache.empty(n, Hkv, D, dt, DEV)
    cache.codes.fill_(0xFF)
    cache.meta.fill_(math.nan)  # what no token has written must not matter
    T = max(max(lens), 1)
    k, v = ((torch.randn(len(lens), T, Hkv, D, generator=_gen(seed + i), device=DEV) * std).to(dt) for i in range(2))
    rfa.kv4_append(cache, k, v, table, _ints([0] * len(lens)), _ints(lens))
    return cache, table, [(quantized(k[b, :n]), quantized(v[b, :n])) for b, n in enumerate(lens)]


def attn_reference(q, values, lens, scale=None, softcap=0.0, slopes=None):
    """(out, bound, lse) of the definition.  Bound: P sc is rounded to 16 bits for its product with the codes, which stand for
    up to 15 sc above the minimum: u sum P (v - min) <= u P (|v| + |min|) <= 2 u max|v| sum P = 2 u vmax, and the result once;
    EXTRA for the fp32 steps: exp2, 1e-6; scores with codes carried as 128 + u, 2^-22 of 128 x 32 |q| sc in each of D / 32
    groups, below 2e-4 of a weight for what is drawn here."""
    B, T, Hq, D = q.shape
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    bound = torch.full_like(out, 1e-6)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        K, V = values[b]
        G = Hq // K.shape[1]
        for h in range(Hq):
            x = q[b, :, h].double() @ K[:, h // G].T * (D ** -0.5 if scale is None else scale)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            ahead = n - T + torch.arange(T, device=DEV)[:, None] - torch.arange(n, device=DEV)[None]
            if slopes is not None:
                x = x - (slopes[b, h] if slopes.dim() == 2 else slopes[h]).double() * ahead
            x = x.masked_fill(ahead < 0, -math.inf)
            lse[b, h] = torch.logsumexp(x, 1)
            P = torch.exp(x - lse[b, h][:, None]).masked_fill(ahead < 0, 0)
            out[b, :, h] = P @ V[:, h // G]
            bound[b, :, h] += (2 * u + 3e-4) * V[:, h // G].abs().max() + 1.01 * u * out[b, :, h].abs()
    return out, bound, lse


def _check(got, lse, ref):
    out, bound, want = ref
    assert torch.isfinite(got).all()
    over = (got.double() - out).abs() / bound
    assert over.max() <= 1, f"{over.max().item():.2f} of the bound at {(over == over.max()).nonzero()[0].tolist()}"
    assert torch.equal(torch.isinf(lse), torch.isinf(want))
    assert ((lse.double() - want).masked_fill(torch.isinf(want), 0)).abs().max() < 1e-3


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_codes_and_values(D, dt):
    """What is appended reads back as the definition says, bit for bit; rows around it stay as they were; ties, constant
    groups, tiny and huge values."""
    import opt_ring_flash_attn_b200 as rfa

    B, T, H = 3, 70, 2
    lens = [200, 70, 130]
    table, n = _table(lens)
    cache = rfa.KV4Cache.empty(n, H, D, dt, DEV)
    cache.codes.zero_()
    cache.meta.zero_()
    k, v = ((torch.randn(B, T, H, D, generator=_gen(i), device=DEV)).to(dt) for i in range(2))
    k[0, 0] = 1.5                                   # a constant group: scale 0
    k[0, 1, :, ::2] = torch.arange(D // 2, device=DEV).to(dt) % 16 / 2   # whole multiples and halves of the scale
    k[0, 1, 0, 0], k[0, 1, 0, 1] = 0, 7.5
    v[1, 2] *= 1e-6
    v[1, 3] *= 1e4
    v[2, 5] = v[2, 5].abs() * 1e-8
    v[2, 6] *= 1e-38  # bf16: scales below the smallest normal number
    start = [130, 0, 60]
    before = cache.codes.clone(), cache.meta.clone()
    rfa.kv4_append(cache, k, v, table, _ints(start))
    gk, gv = rfa.kv4_gather(cache, table, _ints(start), T)
    assert torch.equal(gk, quantized(k).to(dt)) and torch.equal(gv, quantized(v).to(dt))
    # nothing else was written
    mine = torch.zeros(n, 64, dtype=torch.bool, device=DEV)
    for b in range(B):
        for t in range(T):
            pos = start[b] + t
            mine[int(table[b, pos // 64]), pos % 64] = True
    other = ~mine[:, None, None, :].expand(n, H, 2, 64)
    assert torch.equal(cache.codes[other], before[0][other]) and torch.equal(cache.meta[other], before[1][other])
    # a second append elsewhere leaves the first as it is, and strided operands are read as they lie
    fused = torch.randn(B, 5, H * 2 + 1, D, generator=_gen(9), device=DEV).to(dt)
    rfa.kv4_append(cache, fused[:, :, :H], fused[:, :, H + 1:], table, _ints([0, 0, 0]), _ints([5, 0, 5]))
    gk2, _ = rfa.kv4_gather(cache, table, _ints([0, 0, 0]), 5, _ints([5, 0, 3]))
    assert torch.equal(gk2[0], quantized(fused[0, :, :H]).to(dt)) and not gk2[1].any() and not gk2[2, 3:].any()
    assert torch.equal(gk2[2, :3], quantized(fused[2, :3, :H]).to(dt))
    gk3, _ = rfa.kv4_gather(cache, table, _ints(start), T)
    assert torch.equal(gk3[:2], gk[:2])


def test_borders_of_the_table():
    """Positions outside the table, and pages outside the pool, are left out; a group that holds no number reads back as none."""
    import opt_ring_flash_attn_b200 as rfa

    cache = rfa.KV4Cache.empty(3, 1, 64, BF, DEV)
    cache.codes.zero_(), cache.meta.zero_()
    k = torch.randn(1, 64, 1, 64, generator=_gen(0), device=DEV).to(BF)
    for table, start in (([[0, 7]], 64), ([[0, -3]], 64), ([[0, 1]], 128), ([[0, 1]], 2 ** 31 - 32), ([[0, 1]], -64)):
        rfa.kv4_append(cache, k, k, _ints(table), _ints([start]))
        assert not cache.codes.any() and not cache.meta.any()
        gk, gv = rfa.kv4_gather(cache, _ints(table), _ints([start]), 64)
        assert not gk.any() and not gv.any()
    rfa.kv4_append(cache, k, k, _ints([[2, 0]]), _ints([-10]))
    gk, _ = rfa.kv4_gather(cache, _ints([[2, 0]]), _ints([0]), 54)
    assert torch.equal(gk, quantized(k[:, 10:]).to(BF))
    bad = k.clone()
    bad[0, 0, 0, 3], bad[0, 1, 0, 40], bad[0, 2, 0, 5] = math.nan, math.inf, -math.inf
    rfa.kv4_append(cache, bad, bad, _ints([[1]]), _ints([0]))
    gk, _ = rfa.kv4_gather(cache, _ints([[1]]), _ints([0]), 64)
    for t, g in ((0, 0), (1, 1), (2, 0)):
        assert not torch.isfinite(gk[0, t, 0, 32 * g:32 * g + 32]).any()
        assert torch.equal(gk[0, t, 0, 32 * (1 - g):][:32], quantized(k).to(BF)[0, t, 0, 32 * (1 - g):][:32])


LENS = {"one": [1], "zero_and_more": [0, 5, 0, 64, 65], "edges": [63, 128, 129, 16, 17], "long": [3001], "mixed": [2000, 1, 300]}


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("D,dt,Hq,Hkv,T", [(64, BF, 2, 2, 1), (128, BF, 8, 1, 1), (128, HF, 8, 2, 4), (96, HF, 3, 1, 5),
                                           (192, BF, 4, 2, 2), (256, HF, 4, 4, 1), (256, BF, 16, 1, 3), (64, HF, 12, 1, 8),
                                           (128, BF, 5, 5, 20)])
@pytest.mark.parametrize("scores", ["plain", "cap", "bias"])
def test_attention(lens, D, dt, Hq, Hkv, T, scores):
    import opt_ring_flash_attn_b200 as rfa

    lens = LENS[lens]
    cache, table, values = _filled(1, lens, Hkv, D, dt)
    q = torch.randn(len(lens), T, Hq, D, generator=_gen(5), device=DEV).to(dt)
    kw = {}
    if scores != "plain":
        kw["softcap"] = 3.0
    if scores == "bias":
        kw["alibi_slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)
    ref = attn_reference(q, values, lens, softcap=kw.get("softcap", 0.0), slopes=kw.get("alibi_slopes"))
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints(lens), **kw)
    rfa.check("test")
    _check(out, lse, ref)
    assert torch.equal(out, rfa.kv4_attn(q, cache, table, _ints(lens), **kw))  # the same bits every time


def test_many_sequences():
    """More sequences than one warp scans at a time, a few of them long, per-sequence slopes."""
    import opt_ring_flash_attn_b200 as rfa

    lens = [(i * 37) % 200 for i in range(150)]
    lens[70] = 9000
    cache, table, values = _filled(2, lens, 1, 64, BF)
    q = torch.randn(150, 1, 4, 64, generator=_gen(6), device=DEV).to(BF)
    slopes = torch.rand(150, 4, generator=_gen(7), device=DEV) / 16
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints(lens), alibi_slopes=slopes, softmax_scale=0.3)
    rfa.check("test")
    _check(out, lse, attn_reference(q, values, lens, slopes=slopes, scale=0.3))


@pytest.mark.parametrize("peak", ["first", "last", "middle"])
def test_peaked_weights(peak):
    """One key takes nearly all the weight, wherever it stands: the running maximum moves, shared runs are joined."""
    import opt_ring_flash_attn_b200 as rfa

    n = 4000
    cache, table, values = _filled(3, [n], 1, 128, HF, std=0.3)
    at = {"first": 0, "last": n - 1, "middle": n // 2 + 7}[peak]
    q = torch.randn(1, 1, 4, 128, generator=_gen(8), device=DEV).to(HF)
    k = torch.zeros(1, 1, 1, 128, device=DEV, dtype=HF) + q[:, :, :1] * 6
    rfa.kv4_append(cache, k, k, table, _ints([at]))
    values[0][0][at], values[0][1][at] = quantized(k)[0, 0], quantized(k)[0, 0]
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints([n]))
    _check(out, lse, attn_reference(q, values, [n]))


def test_scales_far_apart():
    """V of very different sizes from token to token (the power of two that keeps P sc in fp16 is chosen again on the way), and
    a V that is no number, which reaches its own 32 channels only."""
    import opt_ring_flash_attn_b200 as rfa

    for dt, top in ((BF, 1e20), (HF, 2e3)):
        n = 1000
        table, pool = _table([n])
        cache = rfa.KV4Cache.empty(pool, 1, 128, dt, DEV)
        k = torch.randn(1, n, 1, 128, generator=_gen(1), device=DEV).to(dt)
        v = torch.randn(1, n, 1, 128, generator=_gen(2), device=DEV)
        v[0, :300] /= top
        v[0, 300:310] = 0
        v[0, 500:] *= top / 10
        v = v.to(dt)
        rfa.kv4_append(cache, k, v, table, _ints([0]))
        values = [(quantized(k[0]), quantized(v[0]))]
        q = torch.randn(1, 1, 4, 128, generator=_gen(3), device=DEV).to(dt)
        for m in (n, 700, 310, 305, 5):
            ref = attn_reference(q, [(values[0][0][:m], values[0][1][:m])], [m])
            out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints([m]))
            _check(out, lse, (ref[0], ref[1] * (1 + 1e-6), ref[2]))
        v[0, 400, 0, 40] = math.nan
        rfa.kv4_append(cache, k, v, table, _ints([0]))
        ref = attn_reference(q, values, [n])
        out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints([n]))
        assert out[..., 32:64].isnan().all()
        keep = [c for c in range(128) if not 32 <= c < 64]
        _check(out[..., keep], lse, (ref[0][..., keep], ref[1][..., keep], ref[2]))


def test_bad_pages_and_lengths():
    """A table entry outside the pool: its tokens do not exist.  Lengths beyond the table end at it; negative ones are zero."""
    import opt_ring_flash_attn_b200 as rfa

    lens = [200, 128, 64]
    cache, table, values = _filled(4, lens, 2, 64, BF)
    q = torch.randn(3, 1, 2, 64, generator=_gen(9), device=DEV).to(BF)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = 10 ** 6, -1
    keep = [torch.cat([torch.arange(0, 64), torch.arange(128, 200)]), torch.arange(64, 128), torch.arange(0, 64)]
    out, lse = rfa.kv4_attn_with_lse(q, cache, bad, _ints(lens))
    rfa.check("test")
    part = [(k[i.to(DEV)], v[i.to(DEV)]) for (k, v), i in zip(values, keep)]
    _check(out, lse, attn_reference(q, part, [len(i) for i in keep]))
    out, lse = rfa.kv4_attn_with_lse(q, cache, table[:, :1].contiguous(), _ints([200, 2 ** 31 - 1, -5]))
    rfa.check("test")
    part = [(k[:64], v[:64]) for k, v in values[:2]] + [values[2]]
    _check(out, lse, attn_reference(q, part, [64, 64, 0]))


def test_offsets_beyond_32_bits():
    """Pages whose bytes lie more than 4 GB into the pool."""
    import opt_ring_flash_attn_b200 as rfa

    H, D, n = 8, 256, 40000  # 40000 pages x 8 heads x 16 KB of codes: 5.2 GB
    cache = rfa.KV4Cache(torch.zeros(n, H, 2, 64, D // 2, dtype=torch.uint8, device=DEV),
                         torch.zeros(n, H, 2, 64, D // 32, 2, dtype=BF, device=DEV))
    lens = [100]
    table = _ints([[n - 1, n - 2]])
    k, v = (torch.randn(1, 100, H, D, generator=_gen(i), device=DEV).to(BF) for i in range(2))
    rfa.kv4_append(cache, k, v, table, _ints([0]))
    gk, gv = rfa.kv4_gather(cache, table, _ints([0]), 100)
    assert torch.equal(gk, quantized(k).to(BF)) and torch.equal(gv, quantized(v).to(BF))
    q = torch.randn(1, 1, H, D, generator=_gen(3), device=DEV).to(BF)
    out, lse = rfa.kv4_attn_with_lse(q, cache, table, _ints(lens))
    _check(out, lse, attn_reference(q, [(quantized(k[0]), quantized(v[0]))], lens))
    assert not cache.codes[: n - 2].any()


def test_decoding_step_captured_and_on_two_streams():
    """Append and attend in a captured graph, replayed while the sequences grow; two streams at once."""
    import opt_ring_flash_attn_b200 as rfa

    lens, H, D = [100, 63, 0], 2, 64
    cache, table, values = _filled(5, lens, H, D, BF, spare=1)
    pos = _ints(lens)
    k, v = (torch.zeros(3, 1, H, D, dtype=BF, device=DEV) for _ in range(2))
    q = torch.zeros(3, 1, 2 * H, D, dtype=BF, device=DEV)
    rfa.kv4_attn(q, cache, table, pos)  # sets the device up

    def step():
        rfa.kv4_append(cache, k, v, table, pos)
        pos.add_(1)
        return rfa.kv4_attn_with_lse(q, cache, table, pos, softcap=10.0)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i in range(4):
        for j, t in enumerate((k, v, q)):
            t.copy_(torch.randn(t.shape, generator=_gen(100 + 3 * i + j), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        lens = [n + 1 for n in lens]
        values = [(torch.cat([a, quantized(k[b])]), torch.cat([c, quantized(v[b])])) for b, (a, c) in enumerate(values)]
        _check(out, lse, attn_reference(q, values, lens, softcap=10.0))
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [torch.randn(3, 1, 2 * H, D, generator=_gen(200 + i), device=DEV).to(BF) for i in range(2)]
    torch.cuda.synchronize()
    res = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                res[i].append(rfa.kv4_attn_with_lse(qs[i], cache, table, pos))
    torch.cuda.synchronize()
    for i in range(2):
        for got in res[i]:
            _check(*got, attn_reference(qs[i], values, lens))


def test_prompt_then_tokens():
    """As the operators are used together: a prompt goes through the training operator and into the cache, then tokens are
    decoded; the decoded rows are those of the whole sequence over the cached values, with the same cap and bias."""
    import opt_ring_flash_attn_b200 as rfa

    S, P, Hq, Hkv, D = 300, 290, 4, 2, 128
    x = [torch.randn(1, S, h, D, generator=_gen(300 + i), device=DEV).to(HF) for i, h in enumerate((Hq, Hkv, Hkv))]
    slopes = torch.tensor([2.0 ** (-2 * (h + 1)) for h in range(Hq)], device=DEV)
    kw = dict(softcap=20.0, alibi_slopes=slopes)
    table, n = _table([S])
    cache = rfa.KV4Cache.empty(n, Hkv, D, HF, DEV)
    first = rfa.scored_flash_attn(*(t[:, :P] for t in x), causal=True, **kw)
    assert first.shape == (1, P, Hq, D)
    rfa.kv4_append(cache, x[1][:, :P], x[2][:, :P], table, _ints([0]))
    rows = []
    for i in range(P, S):
        rfa.kv4_append(cache, x[1][:, i:i + 1], x[2][:, i:i + 1], table, _ints([i]))
        rows.append(rfa.kv4_attn(x[0][:, i:i + 1], cache, table, _ints([i + 1]), **kw))
    k, v = rfa.kv4_gather(cache, table, _ints([0]), S)
    whole = rfa.scored_flash_attn(x[0], k, v, causal=True, **kw)
    got, want = torch.cat(rows, 1).double(), whole[:, P:].double()
    # either side rounds its weights and its result (2 u vmax + u vmax); the read-back values are rounded to 16 bits once,
    # u vmax of V, and of K u |q||k| scale < u * 8 of a weight: 8 u vmax
    u, vmax = torch.finfo(HF).eps / 2, v.double().abs().max()
    assert (got - want).abs().max() <= (3 + 3 + 1 + 8) * u * vmax
