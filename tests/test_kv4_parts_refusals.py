"""Arguments of the attention over a part of a cache that are refused (no GPU needed)."""
import ctypes

import pytest
import torch

import opt_ring_flash_attn_b200 as rfa
from opt_ring_flash_attn_b200 import _native

BF = torch.bfloat16


@pytest.mark.parametrize("after", [torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64),
                                   torch.zeros(1, 1, dtype=torch.int32)])
def test_tokens_after(after):
    cache = rfa.KV4Cache.empty(4, 2, 64, BF, device="cpu")
    args = (torch.zeros(1, 1, 4, 64, dtype=BF), cache, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="tokens_after"):
        rfa.kv4_attn_with_lse(*args, tokens_after=after)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rfa.kv4_attn_with_lse(*args, tokens_after=torch.zeros(1, dtype=torch.int32))


def test_abi():
    lib = _native.load()
    st = (ctypes.c_longlong * 3)(64, 64, 64)
    att = lambda Hq=4, after=256, T=1: lib.rfa_kv4_attn_part(  # noqa: E731
        256, st, 256, 256, 4, 256, 2, 256, after, 256, None, 256, 1, T, Hq, 2, 64, 0, 0.1, 0.0, None, 0, 256, None)
    assert att(Hq=3) == -1 and att(after=258) == -1 and att(T=1 << 30) == -5
