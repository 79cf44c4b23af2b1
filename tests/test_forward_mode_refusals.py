"""Forward-mode differentiation is refused by the operators that have no tangents, not dropped (no GPU needed)."""
import pytest
import torch
from torch.autograd import forward_ad

import opt_ring_flash_attn_b200 as rfa
from opt_ring_flash_attn_b200 import scored

BF = torch.bfloat16


@pytest.mark.parametrize("which", ["q", "k", "v", "slopes"])
def test_scored(monkeypatch, which):
    monkeypatch.setattr(scored, "_validate", lambda *a: None)
    x = dict(q=torch.zeros(1, 16, 2, 64, dtype=BF), k=torch.zeros(1, 16, 2, 64, dtype=BF), v=torch.zeros(1, 16, 2, 64, dtype=BF),
             slopes=torch.zeros(2))
    with forward_ad.dual_level():
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                rfa.scored_flash_attn(x["q"], x["k"], x["v"], causal=True, alibi_slopes=x["slopes"])


@pytest.mark.parametrize("which", ["q", "slopes"])
def test_kv4_attn(which):
    cache = rfa.KV4Cache.empty(4, 2, 64, BF, device="cpu")
    x = dict(q=torch.zeros(1, 1, 4, 64, dtype=BF), slopes=torch.zeros(4))
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with forward_ad.dual_level():
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        for f in (rfa.kv4_attn, rfa.kv4_attn_with_lse):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(x["q"], cache, table, lens, alibi_slopes=x["slopes"])
