"""The ring passes of the modified-score attention on CPU tensors: a stand-in for the two hop kernels (fp32 torch) behind the
product's schedules, so that which shard a hop is told it sees, which hops are left out and what travels is checked without a
GPU."""
import ctypes

import pytest
import torch

import fake_kernels
from inproc_ring import InProcRing, drop_workspaces
from opt_ring_flash_attn_b200 import scored

LOG2E = fake_kernels.LOG2E


class Hops:
    """rfa_scored_fwd_hop / rfa_scored_bwd_hop: scores over positions of the whole sequence."""

    def __init__(self, slopes, visible):
        self.slopes, self.visible, self.seen = slopes, visible, []

    def _scores(self, q, k, a):
        S, g = q.shape[1], q.shape[2] // k.shape[2]
        x = (fake_kernels._hf(q) @ fake_kernels._expand(fake_kernels._hf(k), g).transpose(-2, -1)) * a.softmax_scale
        t = torch.tanh(x / a.softcap) if a.softcap else torch.zeros_like(x)
        z = a.softcap * t if a.softcap else x
        qp, kp = (torch.arange(S) + i * S for i in (a.q_shard, a.k_shard))
        z = z - self.slopes[:, None, None] * (qp[:, None] - kp[None]).abs()
        return z.masked_fill(~self.visible[qp][:, kp], float("-inf")), 1 - t * t

    def fwd(self, q, k, v, acc, m, l, out, lse, args, first, last, status, stream=None):
        self.seen.append((args.q_shard, args.k_shard))
        B, S, Hq, D = q.shape
        z, _ = self._scores(q, k, args)
        vh = fake_kernels._expand(fake_kernels._hf(v), Hq // k.shape[2])
        state = acc[: B * Hq * S * D].view(B, Hq, S, D)
        floor = -1e30
        m_old = torch.full((B, Hq, S), floor) if first else m[:, :, :S].clone()
        l_old = torch.zeros(B, Hq, S) if first else l[:, :, :S].clone()
        a_old = torch.zeros(B, Hq, S, D) if first else state.clone()
        m_new = torch.maximum(m_old, z.max(-1).values)
        alpha, p = torch.exp(m_old - m_new), torch.exp(z - m_new[..., None])
        l_new, a_new = l_old * alpha + p.sum(-1), a_old * alpha[..., None] + p @ vh
        if last:
            empty = l_new == 0
            out.copy_((a_new / l_new.masked_fill(empty, 1)[..., None]).transpose(1, 2).to(out.dtype))
            lse[:, :, :S] = (m_new + torch.log(l_new)).masked_fill(empty, float("-inf"))
        else:
            m[:, :, :S], l[:, :, :S] = m_new, l_new
            state.copy_(a_new)

    def bwd(self, q, k, v, dout, lse2, delta, dq_acc, dkdv_out, args, status, stream=None, dq_order=None):
        B, S, Hq, D = q.shape
        Hkv, g = k.shape[2], Hq // k.shape[2]
        z, jac = self._scores(q, k, args)
        l2 = lse2[:, :, :S, None]
        p = torch.exp2(z * LOG2E - l2).masked_fill(torch.isinf(z) | torch.isinf(l2), 0)
        doh, qh = fake_kernels._hf(dout), fake_kernels._hf(q)
        kh, vh = (fake_kernels._expand(fake_kernels._hf(x), g) for x in (k, v))
        ds = p * (doh @ vh.transpose(-2, -1) - delta[:, :, :S, None]) * jac
        dq_acc[: B * Hq * S * D].view(B, Hq, S, D).add_((ds @ kh) * args.softmax_scale)
        for i, x in enumerate(((ds.transpose(-2, -1) @ qh) * args.softmax_scale, p.transpose(-2, -1) @ doh)):
            dkdv_out[i].copy_(x.view(B, Hkv, g, S, D).sum(2).transpose(1, 2))


def _whole(q, k, v, dout, scale, cap, slopes, visible):
    q, k, v = (x.float().requires_grad_(True) for x in (q, k, v))
    g, n = q.shape[2] // k.shape[2], q.shape[1]
    x = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(g, 2)) * scale
    pos = torch.arange(n)
    z = cap * torch.tanh(x / cap) - slopes[:, None, None] * (pos[:, None] - pos[None]).abs()
    empty = ~visible.any(1)
    p = torch.softmax(z.masked_fill(~visible, float("-inf")), -1).masked_fill(empty[:, None], 0)
    out = torch.einsum("bhij,bjhd->bihd", p, v.repeat_interleave(g, 2))
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout.float()))


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("kind", ["causal", "documents", "prefix", "full"])
@pytest.mark.parametrize("wire16", [False, True])
def test_shards_together_are_the_whole(W, kind, wire16, monkeypatch):
    monkeypatch.setenv("OPTIMIZED_RING_BWD_COMM_BF16", "1" if wire16 else "0")
    S, Hq, Hkv, D, scale, cap = 24, 4, 2, 16, 0.3, 4.0
    n = S * W
    g = torch.Generator().manual_seed(W)
    q, k, v, dout = (torch.randn(1, n, h, D, generator=g).bfloat16() for h in (Hq, Hkv, Hkv, Hq))
    slopes = torch.tensor([0.5, 0.1, 0.0, 0.02])
    pos = torch.arange(n)
    doc = (pos >= 10).long() + (pos >= S + 5).long()
    tail = pos >= n - 7
    visible = pos[None] <= pos[:, None] if kind != "full" else torch.ones(n, n, dtype=torch.bool)
    if kind in ("documents", "prefix"):
        if kind == "prefix":  # the first tokens of the second document, from the shard behind as well
            visible = visible | (pos[None] < S + 3)
        visible = visible & (doc[:, None] == doc[None]) & ~tail[:, None] & ~tail[None]
    sees_later = kind in ("prefix", "full")
    hops = Hops(slopes, visible)
    monkeypatch.setattr(scored._native, "scored_fwd_hop", hops.fwd)
    monkeypatch.setattr(scored._native, "scored_bwd_hop", hops.bwd)

    def prepare(out, dout, lse, delta, lse2, dq_acc, status, stream=None):
        fake_kernels.bwd_prepare(out, dout, lse, delta, lse2, dq_acc, status)
        lse2.masked_fill_(lse2 == float("-inf"), float("inf"))

    for name in ("pack_kv", "dq_finalize", "dkdv_accumulate", "dkdv_accumulate_to16", "cast_from_f32"):
        monkeypatch.setattr(scored._Scores, name, staticmethod(getattr(fake_kernels, name)))
    monkeypatch.setattr(scored._Scores, "bwd_prepare", staticmethod(prepare))
    ring = InProcRing(W)

    def one(handle):
        r = handle.ring_rank
        x = [t[:, r * S:(r + 1) * S].contiguous() for t in (q, k, v, dout)]
        sc = scored._Scores(scale, cap, None, kind != "full", None, sees_later, W, r)
        out, lse = scored._forward(handle, *x[:3], sc)
        first = scored._backward(handle, x[3], *x[:3], out, lse, sc.again(), False)
        second = scored._backward(handle, x[3], *x[:3], out, lse, sc.again(), False)  # a pass can be run again
        assert all(torch.equal(a, b) for a, b in zip(first, second))
        return (out, *first)

    try:
        parts = ring.run(one, torch.device("cpu"))
    finally:
        drop_workspaces(ring)
    # hops whose keys all lie behind the queries are left out, and only those
    assert sorted(hops.seen) == [(i, j) for i in range(W) for j in range(W) if sees_later or j <= i]
    for got, want in zip((torch.cat(x, 1) for x in zip(*parts)), _whole(q, k, v, dout, scale, cap, slopes, visible)):
        # rounded to bf16 once, through bf16 at each of W - 1 hops with the 16-bit wire
        assert ((got.float() - want).norm() / want.norm()).item() <= 2.0 ** -8 * (1 + (W if wire16 else 0.1))


def test_arguments_of_a_hop():
    a = scored._Scores(0.5, 3.0, torch.zeros(2, 4), True, torch.zeros(4, dtype=torch.int32), False, 3, 2)
    seen = [(x.q_shard, x.k_shard, x.shards, x.slopes_per_batch, x.causal) for x in (a._next() for _ in range(3))]
    assert seen == [(2, 2, 3, 1, 1), (2, 1, 3, 1, 1), (2, 0, 3, 1, 1)]
    # rfa_score_args: two floats, a pointer, two ints, a pointer, three ints, padded to eight bytes
    assert ctypes.sizeof(type(a.args(0))) == 4 + 4 + 8 + 4 + 4 + 8 + 3 * 4 + 4
