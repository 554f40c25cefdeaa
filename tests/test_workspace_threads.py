"""The default stream's workspaces under threads: two first calls at once get one workspace, and a replaced one stays
allocated (a call in flight may hold its address)."""
import threading
import time

import torch

from src.kernels import hip_paged_attention as hpa


def test_two_first_calls_share_one_workspace(monkeypatch):
    monkeypatch.setattr(hpa, "_workspaces", {})
    monkeypatch.setattr(hpa, "_retired_workspaces", [])
    zeros = torch.zeros

    def slow(*args, **kw):
        time.sleep(0.05)
        return zeros(*args, **kw)

    monkeypatch.setattr(hpa.torch, "zeros", slow)
    for nbytes in (1000, 2 << 20):
        got = []
        threads = [threading.Thread(target=lambda: got.append(hpa._workspace(torch.device("cpu", 0), nbytes, "q4")))
                   for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len({t.data_ptr() for t in got}) == 1
    assert [t.numel() for t in hpa._retired_workspaces] == [1 << 20]
