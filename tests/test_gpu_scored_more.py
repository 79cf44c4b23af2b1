"""Attention with modified scores where the first tests do not reach: hops of a ring that carry a state, at every head dim and kind
of scores, with padding that ends in another rank's shard; long packed rows; tensors beyond 2^31 elements; ordered gradients
without a mask."""
import math

import pytest
import torch

from scored_reference import check, inputs, reference, visible
from test_gpu_scored import BF, DEV, HF, SCORES, _run, _slopes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scores", SCORES)
@pytest.mark.parametrize("kind", ["causal", "docs", "prefix", "full_docs"])
@pytest.mark.parametrize("W,D,dt,deterministic", [(2, 64, HF, False), (3, 96, BF, True), (3, 128, HF, False), (2, 256, BF, False),
                                                  (3, 256, HF, True)])
def test_ring(W, D, dt, deterministic, kind, scores):
    """Shards of 200 rows, two batch rows; the second one's documents begin behind the first shard and end inside the last or the
    one before; what is no document holds no numbers."""
    import opt_ring_flash_attn_b200 as rfa
    from inproc_ring import InProcRing, drop_workspaces
    from opt_ring_flash_attn_b200 import scored

    S, B, Hq, Hkv = 200, 2, 4, 2
    n = S * W
    causal = kind != "full_docs"
    masked = kind != "causal"
    cu = [[0, 150, 160, n - 90, n - 30], [230, 300, 380, 380, 390]]
    pre = [[70, 2, 30, 60], [10, 70, 0, 10]] if kind == "prefix" else None
    sc = dict(SCORES[scores])
    slopes = _slopes(Hq) if sc.pop("bias", False) else None
    q, k, v, dout = inputs(60, B, n, Hq, Hkv, D, dt, DEV)
    vis = visible(n, causal, device=DEV)
    if masked:
        vis = torch.stack([visible(n, causal, cu[b], pre and pre[b], DEV) for b in range(B)])
        for b in range(B):
            real = torch.zeros(n, dtype=torch.bool, device=DEV)
            real[cu[b][0]:cu[b][-1]] = True
            for i, t in enumerate((q, k, v, dout)):
                t[b, ~real] = [math.nan, math.inf, -math.inf, math.nan][i]
    ref = reference(q, k, v, dout, vis, slopes=slopes, **sc)
    ring = InProcRing(W)

    def one(handle):
        sl = slice(handle.ring_rank * S, (handle.ring_rank + 1) * S)
        mask = None
        if masked:
            mask = rfa.document_mask(cu, n, prefix_lens=pre, causal=causal, group=handle, device=DEV).buffer
        x = [t[:, sl].contiguous() for t in (q, k, v, dout)]
        args = (D ** -0.5, sc.get("softcap", 0.0), slopes, causal, mask, kind in ("prefix", "full_docs"), W, handle.ring_rank)
        out, lse = scored._forward(handle, *x[:3], scored._Scores(*args))
        grads = scored._backward(handle, x[3], *x[:3], out, lse, scored._Scores(*args), deterministic)
        return dict(zip(("out", "lse", "dq", "dk", "dv"), (out, lse[:, :, :S], *grads)))

    try:
        parts = ring.run(one, torch.device(DEV))
        torch.cuda.synchronize()
        rfa.check("test")
    finally:
        drop_workspaces(ring)
    check(ref, **{x: torch.cat([p[x] for p in parts], dim=2 if x == "lse" else 1) for x in parts[0]})


def _check_documents(got, q, k, v, dout, cu, pre, slopes, which, **sc):
    """Each document by itself against the definition: the others do not touch it."""
    for d in which:
        a, e = cu[d], cu[d + 1]
        x = [t[:, a:e] for t in (q, k, v, dout)]
        ref = reference(*x, visible(e - a, True, [0, e - a], None if pre is None else [pre[d]], DEV), slopes=slopes, **sc)
        check(ref, **{n: (t[:, :, a:e] if n == "lse" else t[:, a:e]) for n, t in got.items()})


@pytest.mark.parametrize("D,dt,Hq,Hkv", [(64, HF, 4, 2), (128, BF, 4, 1), (256, BF, 2, 2)])
@pytest.mark.parametrize("scores", ["plain", "both"])
def test_long_packed_rows(D, dt, Hq, Hkv, scores):
    """16 000 tokens in documents of 1 to 5000."""
    import opt_ring_flash_attn_b200 as rfa

    S = 16000
    cu = [0, 1, 700, 5700, 5828, 5956, 9000, 12001, 12002, 15500]
    pre = [1, 100, 0, 128, 0, 3044, 17, 0, 1000]
    sc = dict(SCORES[scores])
    slopes = _slopes(Hq) if sc.pop("bias", False) else None
    q, k, v, dout = inputs(61, 1, S, Hq, Hkv, D, dt, DEV)
    mask = rfa.document_mask(cu, S, prefix_lens=pre, device=DEV)
    got = _run(q, k, v, dout, causal=True, mask=mask, alibi_slopes=slopes, **sc)
    for n in got:
        tail = got[n][:, :, cu[-1]:] if n == "lse" else got[n][:, cu[-1]:]
        assert bool((tail == (-math.inf if n == "lse" else 0)).all())
    _check_documents(got, q, k, v, dout, cu, pre, slopes, range(len(pre)), **sc)


def test_tensors_beyond_32_bit_offsets():
    """2^20 tokens of 16 heads of 128: the last documents lie behind element 2^31 of q, out and their gradients."""
    import opt_ring_flash_attn_b200 as rfa

    S, Hq, Hkv, D = 2 ** 20 + 200, 16, 2, 128
    cu = list(range(0, S - 300, 256)) + [S - 300, S - 30]
    assert S * Hq * D > 2 ** 31 + 10 ** 5 and cu[-2] * Hq * D > 2 ** 31 - 10 ** 6
    g = torch.Generator(device=DEV)
    g.manual_seed(62)
    q, dout = (torch.empty(1, S, Hq, D, dtype=BF, device=DEV).normal_(generator=g) for _ in range(2))
    k, v = (torch.empty(1, S, Hkv, D, dtype=BF, device=DEV).normal_(generator=g) for _ in range(2))
    mask = rfa.document_mask(torch.tensor(cu, device=DEV), S)
    for t in (q, k, v):
        t.requires_grad_(True)
    out, lse = rfa.scored_flash_attn_with_lse(q, k, v, causal=True, softcap=20.0, mask=mask)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    rfa.check("test")
    got = dict(out=out.detach(), lse=lse, dq=dq, dk=dk, dv=dv)
    n = len(cu) - 1
    _check_documents(got, q.detach(), k.detach(), v.detach(), dout, cu, None, None, [0, 1, n // 2, n - 3, n - 2, n - 1], softcap=20.0)
    assert not got["out"][:, cu[-1]:].any() and not dq[:, cu[-1]:].any()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("scores", ["plain", "both"])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 1)])
def test_ordered_gradients_repeat(D, causal, scores, Hq, Hkv):
    """Without a mask, K/V tiles shared by several CTAs or not: the same bits every time, and the right ones."""
    sc = dict(SCORES[scores])
    slopes = _slopes(Hq) if sc.pop("bias", False) else None
    q, k, v, dout = inputs(63, 1, 900, Hq, Hkv, D, BF, DEV)
    kw = dict(causal=causal, alibi_slopes=slopes, deterministic=True, **sc)
    got = _run(q, k, v, dout, **kw)
    check(reference(q, k, v, dout, visible(900, causal, device=DEV), slopes=slopes, **sc), **got)
    for _ in range(3):
        again = _run(q, k, v, dout, **kw)
        assert all(torch.equal(got[n], again[n]) for n in got)
