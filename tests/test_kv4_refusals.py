"""Arguments of the 4-bit cache that are refused (no GPU needed)."""
import ctypes

import pytest
import torch

import opt_ring_flash_attn_b200 as rfa
from opt_ring_flash_attn_b200 import _native

BF = torch.bfloat16


def _cache(n=4, H=2, D=64, dt=BF):
    return rfa.KV4Cache.empty(n, H, D, dt, device="cpu")


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_sizes_of_a_cache():
    c = _cache(3, 5, 96, torch.float16)
    assert (c.n_pages, c.n_kv_heads, c.head_dim, c.dtype) == (3, 5, 96, torch.float16)
    assert c.codes.shape == (3, 5, 2, 64, 48) and c.meta.shape == (3, 5, 2, 64, 3, 2)


@pytest.mark.parametrize("D", [0, 32, 80, 160, 512])
def test_head_dims(D):
    with pytest.raises(ValueError, match="head_dim"):
        _cache(D=D)


def test_storage():
    c = _cache()
    for codes, meta in ((c.codes.int(), c.meta), (c.codes[:, :, :1], c.meta), (c.codes, c.meta.float()), (c.codes, c.meta[:2]),
                        (c.codes[:, ::2], c.meta[:, ::2]), (c.codes[:0], c.meta[:0])):
        with pytest.raises(ValueError):
            rfa.KV4Cache(codes, meta)


@pytest.mark.parametrize("change,message", [
    (dict(k=torch.zeros(1, 3, 2, 32, dtype=BF)), "k must be"),
    (dict(v=torch.zeros(1, 3, 1, 64, dtype=BF)), "v must be"),
    (dict(v=torch.zeros(1, 2, 2, 64, dtype=BF)), "differ"),
    (dict(k=torch.zeros(1, 3, 2, 64)), "cache"),
    (dict(block_table=_i32(2, 4)), "block_table"),
    (dict(block_table=_i32(1, 4).long()), "block_table"),
    (dict(positions=_i32(1, 1)), "positions"),
    (dict(counts=_i32(2)), "counts"),
])
def test_append(change, message):
    args = dict(k=torch.zeros(1, 3, 2, 64, dtype=BF), v=torch.zeros(1, 3, 2, 64, dtype=BF), block_table=_i32(1, 4),
                positions=_i32(1), counts=None)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rfa.kv4_append(_cache(), **args)
    with pytest.raises(ValueError, match=message):
        rfa.kv4_append(_cache(), **{**args, **change})


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(1, 1, 3, 64, dtype=BF)), "multiple"),
    (dict(q=torch.zeros(1, 1, 0, 64, dtype=BF)), "multiple"),
    (dict(q=torch.zeros(1, 4, 64, dtype=BF)), "q must be"),
    (dict(lens=_i32(2)), "lens"),
    (dict(softcap=-2.0), "softcap"),
    (dict(softmax_scale=-1.0), "softmax_scale"),
    (dict(alibi_slopes=torch.zeros(5)), "alibi_slopes"),
])
def test_attn(change, message):
    args = dict(q=torch.zeros(1, 1, 4, 64, dtype=BF), block_table=_i32(1, 4), lens=_i32(1))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rfa.kv4_attn(cache=_cache(), **args)
    with pytest.raises(ValueError, match=message):
        rfa.kv4_attn(cache=_cache(), **{**args, **change})
    with pytest.raises(RuntimeError, match="no gradient"):
        rfa.kv4_attn(cache=_cache(), **{**args, "q": args["q"].clone().requires_grad_(True)})


def test_abi_refuses_bad_arguments():
    lib = _native.load()
    st = (ctypes.c_longlong * 3)(64, 64, 64)
    odd = (ctypes.c_longlong * 3)(64, 60, 64)
    app = lambda k=256, s=st, codes=256, n=4, mp=2, T=1, D=64, dt=0: lib.rfa_kv4_append(  # noqa: E731
        k, 256, s, st, codes, 256, n, 256, mp, 256, None, 1, T, 2, D, dt, None)
    assert app(k=None) == -1 and app(k=8) == -1 and app(s=odd) == -1 and app(codes=8) == -1 and app(n=0) == -1
    assert app(mp=0) == -1 and app(T=0) == -1 and app(D=32) == -2 and app(dt=5) == -2 and app(mp=1 << 27) == -5
    att = lambda Hq=4, scale=0.1, cap=0.0, scratch=256, D=64, T=1: lib.rfa_kv4_attn(  # noqa: E731
        256, st, 256, 256, 4, 256, 2, 256, 256, None, scratch, 1, T, Hq, 2, D, 0, scale, cap, None, 0, 256, None)
    assert att(Hq=3) == -1 and att(scale=0.0) == -1 and att(cap=-1.0) == -1 and att(scratch=None) == -1 and att(D=48) == -2
    assert att(T=1 << 30) == -5
    assert lib.rfa_kv4_scratch_elems(1, 1, 4, 3, 64) == 0 and lib.rfa_kv4_scratch_elems(1, 1, 4, 2, 80) == 0
    assert lib.rfa_kv4_scratch_elems(0, 1, 4, 2, 64) == 0
    # two parts of 8 rows per block at least, and a number per unit
    assert lib.rfa_kv4_scratch_elems(5, 1, 4, 2, 128) - lib.rfa_kv4_scratch_elems(4, 1, 4, 2, 128) == 2
    assert lib.rfa_kv4_scratch_elems(1, 1, 4, 2, 128) >= 2 * 148 * 8 * 130


def test_abi_refuses_results_beyond_32_bit_indices():
    """Query rows whose result has more than 2^31 vectors of 16 bytes per sequence."""
    lib = _native.load()
    st = (ctypes.c_longlong * 3)(64, 64, 64)
    rc = lib.rfa_kv4_attn(256, st, 256, 256, 4, 256, 2, 256, 256, None, 256, 1, 1 << 26, 4, 2, 64, 0, 0.1, 0.0, None, 0, 256, None)
    assert rc == -5
