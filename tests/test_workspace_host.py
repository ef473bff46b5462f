"""The workspaces that the wrappers keep (trnrt_amd/kernels/_common.py), on host memory: one for every thread, since a call of
several launches lets another thread's launches in between."""

import threading

import pytest
import torch

from trnrt_amd.kernels import _common as C

DEV = torch.device("cpu", 0)


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    monkeypatch.setattr(C, "stream_ptr", lambda device: 7)
    monkeypatch.setattr(C, "zeroed_workspace", lambda n, device: torch.zeros(n, dtype=torch.uint8))
    monkeypatch.setattr(C, "_WORKSPACES", {})


@pytest.mark.parametrize("keep", ["scratch", "cached_workspace"])
def test_a_thread_has_its_own(host, keep):
    get = getattr(C, keep)
    mine = get(DEV, 1000, "a use of this test")
    theirs = []
    at_once = threading.Barrier(2)

    def other():
        x = get(DEV, 1000, "a use of this test")
        at_once.wait()  # (both alive: a thread's id may be given to a later one)
        theirs.extend((x, get(DEV, 500, "a use of this test")))

    threads = [threading.Thread(target=other) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert get(DEV, 900, "a use of this test") is mine
    assert len({x.data_ptr() for x in (mine, *theirs)}) == 3
    assert get(DEV, 1000, "another use").data_ptr() != mine.data_ptr()
    assert get(DEV, 5000, "a use of this test").numel() >= 5000
