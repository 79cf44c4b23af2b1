"""Arguments of the modified-score attention that are refused, before anything is enqueued (no GPU needed)."""
import pytest
import torch

import opt_ring_flash_attn_b200 as rfa
from opt_ring_flash_attn_b200 import _native, scored


def _qkv(B=1, S=16, H=2, D=64):
    return tuple(torch.zeros(B, S, H, D, dtype=torch.bfloat16) for _ in range(3))


@pytest.mark.parametrize("kw,message", [
    (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("inf")), "softcap"),
    (dict(softcap=1001.0), "softcap"),
    (dict(softcap=float("nan")), "softcap"),
    (dict(softmax_scale=0.0), "softmax_scale"),
    (dict(softmax_scale=float("inf")), "softmax_scale"),
    (dict(alibi_slopes=torch.zeros(3)), "alibi_slopes"),
    (dict(alibi_slopes=torch.zeros(2, dtype=torch.float64)), "float32"),
    (dict(alibi_slopes=torch.zeros(2, requires_grad=True)), "constants"),
    (dict(mask=torch.zeros(4)), "document_mask"),
])
def test_refused(monkeypatch, kw, message):
    # the check for CUDA tensors comes with the checks of shapes; what is behind it is reached without it
    monkeypatch.setattr(scored, "_validate", lambda q, k, v, s: None if s > 0 else _raise("softmax_scale must be positive"))
    with pytest.raises(ValueError, match=message):
        rfa.scored_flash_attn(*_qkv(), **kw)


def _raise(msg):
    raise ValueError(msg)


def test_masks_of_other_calls(monkeypatch):
    monkeypatch.setattr(scored, "_validate", lambda *a: None)
    buf = torch.zeros(8, dtype=torch.int32)
    for mask, causal, message in (
            (rfa.DocumentMask(buf, 1, 16, 1, False, False), True, "causal"),
            (rfa.DocumentMask(buf, 2, 16, 1, True, False), True, "batch"),
            (rfa.DocumentMask(buf, 1, 32, 1, True, False), True, "tokens"),
            (rfa.DocumentMask(buf, 1, 16, 2, True, False), True, "ranks")):
        with pytest.raises(ValueError, match=message):
            rfa.scored_flash_attn(*_qkv(), causal=causal, mask=mask)


@pytest.mark.parametrize("cu,kw,message", [
    ([0, 5, 3, 16], {}, "decrease"),
    ([0, 17], {}, "lie in"),
    ([-1, 16], {}, "lie in"),
    ([0], {}, "cu_seqlens must be"),
    ([0.0, 16.0], {}, "int32"),
    ([[0, 16], [0, 8]], dict(batch=3), "rows"),
    ([0, 16], dict(prefix_lens=[1, 2]), "prefix_lens"),
    ([0, 16], dict(batch=0), "batch"),
])
def test_refused_borders(cu, kw, message):
    with pytest.raises(ValueError, match=message):
        rfa.document_mask(cu, 16, device="cpu", **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rfa.scored_flash_attn(*_qkv(), causal=True)
    with pytest.raises(RuntimeError, match="CUDA only"):
        rfa.document_mask([0, 16], 16, device="cpu")
    with pytest.raises(ValueError, match="multiple"):
        rfa.document_mask([0, 16], 0, device="cpu")


def test_abi_refuses_bad_arguments():
    """The C entry points answer with a code, without touching the device."""
    import ctypes

    lib = _native.load()
    good = dict(softmax_scale=0.1, softcap=0.0, slopes=None, causal=True, mask=None)
    args = lambda **kw: ctypes.byref(_native.score_args(**{**good, **kw}))  # noqa: E731
    fwd = lambda a, q=256, S=128, D=64, dt=0, last=1: lib.rfa_scored_fwd_hop(  # noqa: E731
        q, 256, 256, None, None, None, 256, 256, 1, S, 2, 2, D, dt, a, 1, last, 256, None)
    assert fwd(None) == -1
    assert fwd(args(softmax_scale=0.0)) == -1
    assert fwd(args(softcap=-1.0)) == -1
    assert fwd(args(softcap=2000.0)) == -1
    assert fwd(args(softcap=float("nan"))) == -1
    assert fwd(args(shards=2, q_shard=2)) == -1
    assert fwd(args(shards=0)) == -1
    assert fwd(args(shards=1 << 30), S=128) == -5
    assert fwd(args(), q=None) == -1
    assert fwd(args(), last=0) == -1          # a state is needed
    assert fwd(args(), D=100) == -2
    assert fwd(args(), dt=7) == -2
    a = _native.score_args(**good)
    a.mask = 8                                # not on a 16-byte boundary
    assert fwd(ctypes.byref(a)) == -1
    assert lib.rfa_document_mask(None, None, 1, 1, 1, 16, 1, 1, 256, None) == -1
    assert lib.rfa_document_mask(256, None, 2, 1, 1, 16, 1, 1, 256, None) == -1
    assert lib.rfa_document_mask(256, None, 1, 0, 1, 16, 1, 1, 256, None) == -1
    assert lib.rfa_document_mask(256, None, 1, 1, 1, 16, 1, 1, 8, None) == -1
    assert lib.rfa_mask_elems(0, 16, 1) == 0 and lib.rfa_mask_elems(1, 1 << 30, 4) == 0
    # intervals (4 x S, rounded to 4), hulls (8 per tile), orders (2 per tile, 1 per pair) and 2 borders per row
    assert lib.rfa_mask_elems(2, 300, 1) == 4 * 600 + 10 * 6 + 4 + 4


def test_abi_of_the_shared_rows_refuses_bad_arguments():
    import ctypes

    lib = _native.load()
    good = dict(softmax_scale=0.1, softcap=0.0, slopes=None, causal=True, mask=None)
    args = lambda **kw: ctypes.byref(_native.score_args(**{**good, **kw}))  # noqa: E731
    local = lambda a, q=256, S=4096, D=64, dt=0, scratch=256, H=1, Hkv=1: lib.rfa_scored_fwd_local(  # noqa: E731
        q, 256, 256, 256, 256, scratch, 1, S, H, Hkv, D, dt, a, 0, 256, None)
    assert lib.rfa_scored_fwd_scratch_elems(1, 4096, 1, 64, 1, 0) > 0  # or the calls below do not reach the split
    assert local(None) == -1
    assert local(args(softmax_scale=0.0)) == -1
    assert local(args(), q=None) == -1
    assert local(args(), scratch=264) == -1   # not on a 16-byte boundary
    assert local(args(), Hkv=2) == -1
    assert local(args(), S=0) == -1
    assert local(args(), D=100) == -2
    assert local(args(), dt=7) == -2
    assert lib.rfa_scored_fwd_scratch_elems(1, 4096, 1, 100, 1, 0) == 0
    assert lib.rfa_scored_fwd_scratch_elems(0, 4096, 1, 64, 1, 0) == 0
    # one head of 64 over 4096 rows: copies of the state, each O, maxima and sums
    assert lib.rfa_scored_fwd_scratch_elems(1, 4096, 1, 64, 1, 0) % (4096 * 66) == 0
    # many heads, or documents that are short on average: one launch
    assert lib.rfa_scored_fwd_scratch_elems(1, 4096, 32, 128, 1, 0) == 0
    assert lib.rfa_scored_fwd_scratch_elems(1, 4096, 1, 64, 1, 200) == 0
