"""Scales and caps whose quotient leaves fp32 (a score of 0 would become 0 times infinity) are refused."""
import ctypes

import pytest
import torch

import opt_ring_flash_attn_b200 as rfa
from opt_ring_flash_attn_b200 import _native, scored

BF = torch.bfloat16
BAD = [(dict(softcap=1e-40), "softcap"), (dict(softcap=1.0, softmax_scale=2e38), "softcap"),
       (dict(softmax_scale=2.9e38), "softmax_scale"), (dict(softmax_scale=1e300), "softmax_scale")]


@pytest.mark.parametrize("kw,message", BAD)
def test_refused(monkeypatch, kw, message):
    monkeypatch.setattr(scored, "_validate", lambda *a: None)
    x = torch.zeros(1, 16, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match=message):
        rfa.scored_flash_attn(x, x, x, **kw)
    cache = rfa.KV4Cache.empty(4, 2, 64, BF, device="cpu")
    with pytest.raises(ValueError, match=message):
        rfa.kv4_attn(x[:, :1], cache, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), **kw)


def test_abi():
    lib = _native.load()
    st = (ctypes.c_longlong * 3)(64, 64, 64)
    for scale, cap in ((0.1, 1e-40), (2e38, 1.0), (2.9e38, 0.0)):
        a = ctypes.byref(_native.score_args(scale, cap, None, True, None))
        assert lib.rfa_scored_fwd_hop(256, 256, 256, None, None, None, 256, 256, 1, 128, 2, 2, 64, 0, a, 1, 1, 256, None) == -1
        assert lib.rfa_kv4_attn(256, st, 256, 256, 4, 256, 2, 256, 256, None, 256, 1, 1, 4, 2, 64, 0, scale, cap, None, 0, 256,
                                None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 256])
def test_smallest_caps(D):
    """The smallest caps that are taken: scores of 0 stay 0, all weights are even."""
    dev = torch.device("cuda", 0)
    S = 200
    q = torch.zeros(1, S, 2, D, dtype=BF, device=dev)
    q[0, 100:] = 1
    v = torch.ones_like(q)
    for cap in (2e-38, 1e-30):
        out = rfa.scored_flash_attn(q, q, v, causal=True, softcap=cap, softmax_scale=0.125)
        assert torch.equal(out, v)
