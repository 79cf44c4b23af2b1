"""What the backward pass of the modified-score attention needs and what was changed in place since the forward pass (no GPU
needed: the passes themselves are replaced)."""
import pytest
import torch

import opt_ring_flash_attn_b200 as rfa
from opt_ring_flash_attn_b200 import _native, scored

S, H, D = 16, 2, 64


@pytest.fixture
def passes(monkeypatch):
    monkeypatch.setattr(scored, "_validate", lambda *a: None)
    monkeypatch.setattr(scored, "_forward", lambda g, q, k, v, sc: (torch.zeros_like(q), torch.zeros(1, H, 128)))
    monkeypatch.setattr(scored, "_backward", lambda g, do, q, k, v, *a: (torch.ones_like(q), torch.ones_like(k), torch.ones_like(v)))
    monkeypatch.setattr(_native, "document_mask", lambda *a, **k: None)


def _call(slopes, mask):
    q, k, v = (torch.zeros(1, S, H, D, dtype=torch.bfloat16, requires_grad=True) for _ in range(3))
    return q, rfa.scored_flash_attn(q, k, v, causal=True, alibi_slopes=slopes, mask=mask)


def _mask():
    return rfa.DocumentMask(torch.zeros(64, dtype=torch.int32), 1, S, 1, True, False)


def test_nothing_changed(passes):
    q, out = _call(torch.ones(H), _mask())
    out.sum().backward()
    assert bool((q.grad == 1).all())
    q, out = _call(None, None)
    out.sum().backward()
    assert bool((q.grad == 1).all())


def test_slopes_changed(passes):
    slopes = torch.ones(H)
    _, out = _call(slopes, None)
    slopes.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_mask_updated(passes):
    mask = _mask()
    _, out = _call(None, mask)
    mask.update_([0, 5, S])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    q, out = _call(None, mask)  # and a call after the update is in order
    out.sum().backward()
    assert bool((q.grad == 1).all())


def test_made_in_inference_mode(passes):
    with torch.inference_mode():
        mask, slopes = _mask(), torch.ones(H)
        mask.update_([0, S])
    q, out = _call(slopes, mask)
    out.sum().backward()
    assert bool((q.grad == 1).all())
