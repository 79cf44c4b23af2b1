"""Borders and prefixes of document masks that int32 does not hold."""
import pytest
import torch

import opt_ring_flash_attn_b200 as rfa
from opt_ring_flash_attn_b200 import scored


def test_large_numbers_stay_on_their_side():
    big = torch.tensor([-2 ** 40, -1, 0, 7, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 62])
    got = scored._int32(big, torch.device("cpu"), "cu_seqlens")
    assert got.dtype == torch.int32 and got.tolist() == [-1, -1, 0, 7] + [2 ** 31 - 1] * 4
    assert scored._int32([0, 2 ** 33], torch.device("cpu"), "prefix_lens").tolist() == [0, 2 ** 31 - 1]


@pytest.mark.gpu
def test_masks_of_large_numbers():
    dev, S = torch.device("cuda", 0), 300
    want = rfa.document_mask([0, 100, 300], S, prefix_lens=[100, 0], device=dev)
    got = rfa.document_mask(torch.tensor([-2 ** 33, 100, 2 ** 32 + 5], device=dev), S,
                            prefix_lens=torch.tensor([2 ** 32 + 3, -2 ** 40], device=dev))
    assert torch.equal(got.buffer, want.buffer)
    assert torch.equal(rfa.document_mask([0, 100, 300], S, prefix_lens=[2 ** 40, 0], device=dev).buffer, want.buffer)


def test_device_without_a_number(monkeypatch):
    """``device="cuda"`` is the current device, also for borders that lie there already."""
    seen = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(scored, "_borders", lambda cu, pre, b, s, device: seen.append(device) or (cu, pre))
    monkeypatch.setattr(scored._native, "mask_elems", lambda *a: (_ for _ in ()).throw(StopIteration))
    with pytest.raises(StopIteration):
        rfa.document_mask(torch.tensor([0, 16]), 16, device="cuda")
    assert seen == [torch.device("cuda", 3)]


@pytest.mark.gpu
def test_borders_on_the_current_device():
    mask = rfa.document_mask(torch.tensor([0, 100, 300], device="cuda"), 300, device="cuda")
    assert mask.device == torch.device("cuda", torch.cuda.current_device())


def test_typical_keys_of_many_documents():
    """More borders than tokens (rows padded to a fixed number of documents): short documents, not one long one."""
    assert scored._typical_keys(1000, 1) == 1000 and scored._typical_keys(1000, 10) == 200
    assert scored._typical_keys(1000, 5000) == 1
