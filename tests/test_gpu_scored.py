"""Attention with modified scores against its definition in 64 bits: caps, distance bias, document and prefix masks, both
directions, types and head layouts; then the ways it is called (ring, streams, graphs, padding that holds anything)."""
import math

import pytest
import torch

from scored_reference import check, inputs, reference, visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def _slopes(H, signed=False):
    s = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEV)
    return -s / 16 if signed else s


def _run(q, k, v, dout, deterministic=False, **kw):
    import opt_ring_flash_attn_b200 as rfa

    q, k, v = (x.detach().clone().requires_grad_(True) for x in (q, k, v))
    with rfa.deterministic(deterministic):
        out, lse = rfa.scored_flash_attn_with_lse(q, k, v, **kw)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    rfa.check("test")
    return dict(out=out.detach(), lse=lse, dq=dq, dk=dk, dv=dv)


SCORES = {"plain": {}, "bias": dict(bias=True), "cap": dict(softcap=20.0), "both": dict(bias=True, softcap=30.0)}
SHAPES = [  # B, S, Hq, Hkv, D, dtype
    (1, 1, 1, 1, 64, BF), (2, 7, 4, 2, 64, HF), (1, 128, 2, 1, 128, BF), (1, 129, 4, 4, 32, HF), (2, 300, 4, 1, 128, HF),
    (1, 513, 2, 2, 96, BF), (1, 200, 2, 1, 256, BF), (2, 333, 2, 2, 160, HF), (1, 700, 8, 2, 64, BF), (1, 640, 2, 2, 256, HF),
    (1, 260, 3, 1, 8, BF),
]


@pytest.mark.parametrize("scores", SCORES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:5])))
def test_scores(shape, causal, scores):
    B, S, Hq, Hkv, D, dt = shape
    sc = dict(SCORES[scores])
    slopes = _slopes(Hq) if sc.pop("bias", False) else None
    q, k, v, dout = inputs(1, B, S, Hq, Hkv, D, dt, DEV, std=1.5)
    ref = reference(q, k, v, dout, visible(S, causal, device=DEV), slopes=slopes, **sc)
    check(ref, **_run(q, k, v, dout, causal=causal, alibi_slopes=slopes, **sc))


DOCS = {  # borders per batch row (repeated to B), prefixes
    "two": ([0, 130, 400], [50, 200]),
    "one_row_docs": ([0, 1, 2, 3, 130, 131, 400], [0, 1, 0, 127, 1, 300]),
    "tail": ([0, 100, 100, 270], [10, 0, 170]),
    "offset_begin": ([37, 200, 390], [163, 5]),
    "nothing": ([0, 0], [0]),
    "only_middle": ([150, 160], [3]),
    "tiles": ([0, 128, 256, 400], [128, 0, 64]),
}


@pytest.mark.parametrize("scores", ["plain", "both"])
@pytest.mark.parametrize("kind", ["causal", "prefix", "full"])
@pytest.mark.parametrize("docs", DOCS)
@pytest.mark.parametrize("D,dt,Hkv", [(64, BF, 2), (128, HF, 1), (256, BF, 2)])
def test_documents(docs, kind, scores, D, dt, Hkv):
    import opt_ring_flash_attn_b200 as rfa

    S, Hq = 400, 2
    cu, prefix = DOCS[docs]
    prefix = prefix if kind == "prefix" else None
    causal = kind != "full"
    sc = dict(SCORES[scores])
    slopes = _slopes(Hq) if sc.pop("bias", False) else None
    q, k, v, dout = inputs(2, 1, S, Hq, Hkv, D, dt, DEV)
    ref = reference(q, k, v, dout, visible(S, causal, cu, prefix, DEV), slopes=slopes, **sc)
    mask = rfa.document_mask(cu, S, prefix_lens=prefix, causal=causal, device=DEV)
    # rows that belong to no document may hold anything
    real = torch.zeros(S, dtype=torch.bool, device=DEV)
    real[cu[0]:cu[-1]] = True
    for i, t in enumerate((q, k, v, dout)):
        t[:, ~real] = [math.nan, math.inf, -math.inf, math.nan][i]
    check(ref, **_run(q, k, v, dout, causal=causal, mask=mask, alibi_slopes=slopes, **sc))


@pytest.mark.parametrize("D,dt", [(64, HF), (128, BF), (256, HF)])
@pytest.mark.parametrize("deterministic", [False, True])
def test_documents_per_row(D, dt, deterministic):
    """Batch rows with documents of their own, head groups, more key tiles than one; ordered gradients repeat bit for bit."""
    import opt_ring_flash_attn_b200 as rfa

    B, S, Hq, Hkv = 3, 900, 4, 2
    cu = [[0, 300, 800, 880], [0, 900, 900, 900], [5, 6, 450, 890]]
    pre = [[100, 3, 0], [400, 0, 0], [0, 444, 20]]
    q, k, v, dout = inputs(3, B, S, Hq, Hkv, D, dt, DEV)
    slopes = torch.stack([_slopes(Hq), _slopes(Hq, signed=True), 0 * _slopes(Hq)])
    vis = torch.stack([visible(S, True, c, p, DEV) for c, p in zip(cu, pre)])
    ref = reference(q, k, v, dout, vis, slopes=slopes, softcap=25.0)
    mask = rfa.document_mask(torch.tensor(cu, device=DEV), S, prefix_lens=torch.tensor(pre, device=DEV))
    kw = dict(causal=True, mask=mask, alibi_slopes=slopes, softcap=25.0, deterministic=deterministic)
    got = _run(q, k, v, dout, **kw)
    check(ref, **got)
    if deterministic:
        again = _run(q, k, v, dout, **kw)
        assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("value,cap", [(1e-3, 5.0), (0.6, 5.0), (1.0, 5.0), (4.0, 5.0), (1e4, 5.0), (1.0, 1000.0), (4.0, 0.01)])
def test_cap_over_its_whole_range(D, value, cap):
    """Scores far below the cap, around it (where one route to the tanh hands over to the other) and far beyond it (where it
    is 1 and nothing flows back); the largest cap and a tiny one."""
    q, k, v, dout = inputs(4, 1, 700, 2, 2, D, HF, DEV, std=math.sqrt(value))
    ref = reference(q, k, v, dout, visible(700, True, device=DEV), softcap=cap)
    check(ref, **_run(q, k, v, dout, causal=True, softcap=cap))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_outliers_beyond_the_cap(D):
    """A few scores beyond the cap among ordinary ones, at the start, inside and at the end of a tile, in one head of two."""
    S = 520
    q, k, v, dout = inputs(15, 1, S, 2, 1, D, BF, DEV)
    q[0, [5, 200, 519], 1] *= 30
    k[0, [0, 127, 128, 300], 0] *= 20
    ref = reference(q, k, v, dout, visible(S, True, device=DEV), softcap=15.0)
    check(ref, **_run(q, k, v, dout, causal=True, softcap=15.0))


def test_gradient_against_differences():
    """The gradients are those of the function that the forward pass computes: directional differences in fp64 of the
    definition, which the forward pass is checked against above."""
    import opt_ring_flash_attn_b200 as rfa

    S, H, D, cap = 150, 2, 64, 10.0
    cu, pre = [0, 60, 150], [20, 10]
    q, k, v, dout = inputs(5, 1, S, H, H, D, HF, DEV, std=2.0)
    slopes = _slopes(H)
    vis = visible(S, True, cu, pre, DEV)
    mask = rfa.document_mask(cu, S, prefix_lens=pre, device=DEV)
    got = _run(q, k, v, dout, causal=True, mask=mask, alibi_slopes=slopes, softcap=cap)
    ref = reference(q, k, v, dout, vis, slopes=slopes, softcap=cap)

    def loss(qq, kk, vv):
        total = 0.0
        pos = torch.arange(S, device=DEV, dtype=torch.float64)
        for h in range(H):
            x = cap * torch.tanh(qq[0, :, h] @ kk[0, :, h].T * D ** -0.5 / cap)
            x = x - slopes[h].double() * (pos[:, None] - pos[None]).abs()
            total += (torch.softmax(x.masked_fill(~vis, -math.inf), 1) @ vv[0, :, h] * dout[0, :, h].double()).sum()
        return total

    g = torch.Generator(device=DEV)
    g.manual_seed(0)
    base = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(base[i].shape, generator=g, device=DEV, dtype=torch.float64)
        eps = 1e-4
        ends = [loss(*[t + (s * eps * d if j == i else 0) for j, t in enumerate(base)]) for s in (1, -1)]
        slope = ((ends[0] - ends[1]) / (2 * eps)).item()
        # what the elementwise bound allows in this direction; the differences themselves are off by eps^2
        allowed = (ref[name][1] * d.abs()).sum().item() + 1e-4 * abs(slope)
        assert abs((got[name].double() * d).sum().item() - slope) <= allowed


@pytest.mark.parametrize("W", [2, 3])
@pytest.mark.parametrize("kind", ["causal", "docs", "prefix", "full_docs"])
@pytest.mark.parametrize("deterministic", [False, True])
def test_ring(W, kind, deterministic):
    """All ranks of a ring in one process: the shards together give what the whole sequence gives."""
    import opt_ring_flash_attn_b200 as rfa
    from inproc_ring import InProcRing, drop_workspaces

    S, Hq, Hkv, D, dt = 200, 4, 2, 64, BF
    n = S * W
    cu, pre = [0, 150, 160, n - 90, n - 30], [70, 2, 30, 60]
    causal = kind != "full_docs"
    q, k, v, dout = inputs(6, 1, n, Hq, Hkv, D, dt, DEV)
    slopes = _slopes(Hq)
    docs = dict(cu=cu, prefix=pre if kind == "prefix" else None) if kind != "causal" else {}
    ref = reference(q, k, v, dout, visible(n, causal, device=DEV, **docs), slopes=slopes, softcap=15.0)
    ring = InProcRing(W)

    def one(handle):
        # the passes themselves: one engine thread per device runs all backward passes of autograd, and here the ranks wait
        # for one another
        from opt_ring_flash_attn_b200 import scored

        sl = slice(handle.ring_rank * S, (handle.ring_rank + 1) * S)
        mask = None
        if kind != "causal":
            mask = rfa.document_mask(cu, n, prefix_lens=docs["prefix"], causal=causal, group=handle, device=DEV).buffer
        x = [t[:, sl].contiguous() for t in (q, k, v, dout)]
        args = (D ** -0.5, 15.0, slopes, causal, mask, kind in ("prefix", "full_docs"), W, handle.ring_rank)
        out, lse = scored._forward(handle, *x[:3], scored._Scores(*args))
        grads = scored._backward(handle, x[3], *x[:3], out, lse, scored._Scores(*args), deterministic)
        return dict(zip(("out", "lse", "dq", "dk", "dv"), (out, lse[:, :, :S], *grads)))

    try:
        parts = ring.run(one, torch.device(DEV))
        torch.cuda.synchronize()
        rfa.check("test")
    finally:
        drop_workspaces(ring)
    got = {x: torch.cat([p[x] for p in parts], dim=2 if x == "lse" else 1) for x in parts[0]}
    check(ref, **got)


def test_graph_and_mask_update():
    """A captured step replayed on other inputs and other documents."""
    import opt_ring_flash_attn_b200 as rfa

    S, H, D = 300, 2, 64
    q, k, v, dout = inputs(7, 1, S, H, H, D, BF, DEV)
    borders = torch.tensor([0, 100, 300], device=DEV, dtype=torch.int32)
    mask = rfa.document_mask(borders, S)
    sq, sk, sv = (x.clone().requires_grad_(True) for x in (q, k, v))

    def step():
        mask.update_(borders)
        out = rfa.scored_flash_attn(sq, sk, sv, causal=True, softcap=10.0, mask=mask)
        return (out.detach(), *torch.autograd.grad(out, (sq, sk, sv), dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        got2 = step()
    for seed, cu in ((8, [0, 10, 290]), (9, [3, 250, 300])):
        q2, k2, v2, _ = inputs(seed, 1, S, H, H, D, BF, DEV)
        with torch.no_grad():
            sq.copy_(q2), sk.copy_(k2), sv.copy_(v2)
        borders.copy_(torch.tensor(cu))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        ref = reference(q2, k2, v2, dout, visible(S, True, cu, device=DEV), softcap=10.0)
        for g in (got, got2):
            check(ref, **dict(zip(("out", "dq", "dk", "dv"), g)))


def test_streams_strides_and_offsets():
    """Passes on two streams at once; operands that are slices of larger tensors, off the 16-byte boundary, or expanded."""
    import opt_ring_flash_attn_b200 as rfa

    S, H, D = 700, 4, 64
    sets = [inputs(10 + i, 1, S, H, H, D, BF, DEV) for i in range(2)]
    refs = [reference(*s, visible(S, True, device=DEV), softcap=10.0) for s in sets]
    torch.cuda.synchronize()
    streams, res = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                res[i].append(_run_async(rfa, *sets[i], causal=True, softcap=10.0))
    torch.cuda.synchronize()
    for i in range(2):
        for got in res[i]:
            check(refs[i], **got)
    q, k, v, dout = sets[0]
    qkv = torch.stack([q, k, v], 2)
    got = _run(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], dout, causal=True, softcap=10.0)
    check(refs[0], **got)
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view_as(q)
    off.copy_(q)
    check(refs[0], out=rfa.scored_flash_attn(off, k, v, causal=True, softcap=10.0))
    leaf = q.clone().requires_grad_(True)
    rfa.scored_flash_attn(leaf, k, v, causal=True, softcap=10.0).sum().backward()  # an expanded gradient
    ref1 = reference(q, k, v, torch.ones_like(dout), visible(S, True, device=DEV), softcap=10.0)
    check(ref1, dq=leaf.grad)


def _run_async(rfa, q, k, v, dout, **kw):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out, lse = rfa.scored_flash_attn_with_lse(q, k, v, **kw)
    return dict(zip(("out", "lse", "dq", "dk", "dv"), (out.detach(), lse, *torch.autograd.grad(out, (q, k, v), dout))))


def test_plain_scores_and_no_mask_agree_with_ring_flash_attn():
    import opt_ring_flash_attn_b200 as rfa

    q, k, v, dout = inputs(12, 2, 500, 4, 2, 128, BF, DEV)
    for causal in (True, False):
        base, lse = rfa.ring_flash_attn_with_lse(q, k, v, causal=causal)
        out, lse2 = rfa.scored_flash_attn_with_lse(q, k, v, causal=causal)
        assert torch.equal(base, out) and torch.equal(lse, lse2)


def test_baseline_style_call_takes_slopes():
    import opt_ring_flash_attn_b200 as rfa

    q, k, v, dout = inputs(13, 1, 200, 4, 2, 64, BF, DEV)
    slopes = _slopes(4)
    out = rfa.ring_flash_attn_func(q, k, v, causal=True, alibi_slopes=slopes)
    assert torch.equal(out, rfa.scored_flash_attn(q, k, v, causal=True, alibi_slopes=slopes))
    out2, lse, probs = rfa.ring_flash_attn_func(q, k, v, causal=True, alibi_slopes=slopes, return_attn_probs=True)
    assert torch.equal(out, out2) and lse.shape == (1, 4, 200) and probs is None


def test_empty_calls():
    import opt_ring_flash_attn_b200 as rfa

    for shape in ((0, 16, 2, 64), (1, 0, 2, 64)):
        q = torch.zeros(shape, dtype=BF, device=DEV, requires_grad=True)
        out = rfa.scored_flash_attn(q, q, q, causal=True)
        out.sum().backward()
        assert out.shape == shape and q.grad.shape == shape


def test_malformed_borders_on_the_device_are_safe():
    """Borders that fall, or lie outside the sequence: some mask, but no access outside the tensors (the intervals are
    clamped; every loop of the kernels runs over tiles of the block) and no wait that does not end."""
    import opt_ring_flash_attn_b200 as rfa

    S = 300
    q, k, v, dout = inputs(14, 1, S, 2, 2, 64, BF, DEV)
    for cu in ([0, 500, 100, 300], [-50, 200, 1000], [300, 200, 100, 0]):
        mask = rfa.document_mask(torch.tensor(cu, device=DEV), S, prefix_lens=torch.tensor([1000] * (len(cu) - 1), device=DEV))
        got = _run(q, k, v, dout, causal=True, mask=mask)  # ends with a check of the status word
        assert got["out"].shape == q.shape


SPLIT = [  # B, S, Hq, Hkv, D, dtype, causal, scores, borders, prefixes
    (1, 2053, 2, 1, 64, BF, True, "both", None, None),
    (1, 2500, 1, 1, 128, HF, False, "plain", None, None),
    (2, 2300, 2, 2, 256, BF, True, "cap", None, None),
    (1, 2048, 3, 1, 40, HF, False, "bias", None, None),
    (1, 3000, 2, 2, 96, BF, True, "both", [7, 2900], [1200]),
    # the second tile of a pair sees far more than the first; runs of key tiles that no row of a pair sees; padding only
    (1, 3900, 2, 1, 64, HF, False, "plain", [0, 130, 3300], None),
    (1, 3900, 1, 1, 128, BF, True, "cap", [300, 3500, 3600], [5, 90]),
]


@pytest.mark.parametrize("case", SPLIT, ids=lambda c: "-".join(map(str, c[1:5])) + "-" + c[7])
def test_rows_shared_by_ctas(case):
    """Few heads: the key tiles of a row are shared by several CTAs, whose states are joined."""
    import opt_ring_flash_attn_b200 as rfa
    from opt_ring_flash_attn_b200 import _native

    B, S, Hq, Hkv, D, dt, causal, scores, cu, pre = case
    sc = dict(SCORES[scores])
    slopes = _slopes(Hq, signed=causal) if sc.pop("bias", False) else None
    q, k, v, dout = inputs(16, B, S, Hq, Hkv, D, dt, DEV, std=1.5)
    ref = reference(q, k, v, dout, visible(S, causal, cu, pre, DEV), slopes=slopes, **sc)
    mask, typical = None, 0
    if cu is not None:
        mask = rfa.document_mask(cu, S, prefix_lens=pre, causal=causal, device=DEV)
        typical = mask.typical_keys
        real = torch.zeros(S, dtype=torch.bool, device=DEV)
        real[cu[0]:cu[-1]] = True
        for i, t in enumerate((q, k, v, dout)):
            t[:, ~real] = [math.nan, math.inf, -math.inf, math.nan][i]
    assert _native.scored_fwd_scratch_elems(B, S, Hq, D, causal, typical) > 0  # or the case tests nothing
    got = _run(q, k, v, dout, causal=causal, mask=mask, alibi_slopes=slopes, **sc)
    check(ref, **got)
    again = _run(q, k, v, dout, causal=causal, mask=mask, alibi_slopes=slopes, **sc)
    assert torch.equal(got["out"], again["out"]) and torch.equal(got["lse"], again["lse"])


def test_no_number_reaches_its_row_from_any_share():
    """A score that is no number makes its row NaN, whichever CTA meets it, and no other row."""
    import opt_ring_flash_attn_b200 as rfa

    S = 2100
    q, k, v, _ = inputs(17, 1, S, 1, 1, 64, BF, DEV)
    q[0, 2000, 0, 3] = math.nan
    out, lse = rfa.scored_flash_attn_with_lse(q, k, v, causal=True)
    rfa.check("test")
    bad = torch.zeros(S, dtype=torch.bool, device=DEV)
    bad[2000] = True
    assert torch.equal(out.isnan().all(-1).flatten(), bad) and torch.equal(out.isnan().any(-1).flatten(), bad)
    assert torch.equal(lse.isnan().flatten(), bad)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_beyond_the_cap_beside_padding_that_is_no_number(D):
    """Keys whose scores lie beyond the cap share a run of 32 keys with padding of NaN: their tanh is still exact."""
    import opt_ring_flash_attn_b200 as rfa

    S, end = 400, 330
    q, k, v, dout = inputs(18, 1, S, 2, 1, D, BF, DEV)
    k[0, end - 6:end] *= 30  # these only: a tile with many such scores would change the route of the next ones
    ref = reference(q, k, v, dout, visible(S, False, [0, end], None, DEV), softcap=15.0)
    mask = rfa.document_mask([0, end], S, causal=False, device=DEV)
    for t in (q, k, v, dout):
        t[:, end:] = math.nan
    check(ref, **_run(q, k, v, dout, mask=mask, softcap=15.0))
