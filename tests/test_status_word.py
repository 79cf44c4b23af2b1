"""The status word of the operators that allocate their scratch per call (no GPU needed)."""
import threading
import time

import torch

from opt_ring_flash_attn_b200 import workspace


def test_first_calls_of_two_threads_share_the_word(monkeypatch):
    monkeypatch.setattr(workspace, "_status_cache", {})
    new = workspace._new_status

    def slowly(device):
        time.sleep(0.05)
        return new(device)

    monkeypatch.setattr(workspace, "_new_status", slowly)
    got = []
    threads = [threading.Thread(target=lambda: got.append(workspace.status_workspace(torch.device("cpu")))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and all(ws is got[0] for ws in got)


def test_the_word_outlives_the_scratch():
    """A captured decoding step is replayed after ``shutdown()``: its kernels read the word they were captured with."""
    ws = workspace.status_workspace(torch.device("cpu"))
    workspace.clear()
    assert workspace.status_workspace(torch.device("cpu")) is ws
