"""Scratch of the Python face: what a call is given while another one's kernels may still be queued."""
import threading

import pytest
import torch


def in_threads(n, work):
    """work() on n threads that are all alive at once; their results."""
    got, meet = [None] * n, threading.Barrier(n, timeout=60)

    def one(i):
        meet.wait()
        got[i] = work()
        meet.wait()

    threads = [threading.Thread(target=one, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return got


@pytest.fixture
def ops(monkeypatch):
    from tessera_b200 import ops
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_q8_scratch", {})
    return ops


def test_threads_on_one_stream_have_scratch_of_their_own(ops):
    """A call's kernels meet in its scratch, and the library is called without the interpreter's lock: with one buffer for
    two threads, one's second kernel can read what the other's first one left."""
    like = torch.zeros(1)
    for work in (lambda: ops._scratch(100, 0, 7, like)[0], lambda: ops.workspace(100, "cpu").data_ptr()):
        got = in_threads(4, work)
        assert len(set(got)) == 4


def test_a_thread_keeps_its_scratch_and_streams_do_not_share(ops):
    like = torch.zeros(1)
    first, owner = ops._scratch(100, 0, 7, like)
    assert ops._scratch(200, 0, 7, like)[0] == first
    assert ops._scratch(100, 0, 8, like)[0] != first and ops._scratch(100, 1, 7, like)[0] != first
    grown, larger = ops._scratch(owner.numel() + 1, 0, 7, like)
    assert larger.numel() > owner.numel() and ops._scratch(100, 0, 7, like)[0] == grown
    assert ops._scratch(0, 0, 7, like) == (None, None)


def test_workspace_sizes_are_kept_by_device(ops, monkeypatch):
    """A size goes by the current device's multiprocessors."""
    class Library:
        count = 0

        def ts_size(self, rows, keys):
            self.count += 1
            return self.count

    monkeypatch.setattr(ops, "lib", Library())
    ops._q8_workspace.cache_clear()
    try:
        assert [ops._q8_workspace("ts_size", dev, 5, 6) for dev in (0, 1, 0, 1)] == [1, 2, 1, 2]
    finally:
        ops._q8_workspace.cache_clear()


def test_captured_calls_have_scratch_of_their_own(ops, monkeypatch):
    """A graph keeps the addresses that its calls had: scratch shared with another graph, or with calls that may need more of
    it later, would be written by both, or be somebody else's by then."""
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
    made, empty = [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda *shape, device=None, **more: made.append(device) or empty(*shape, **more))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: type("Stream", (), {"cuda_stream": 7}))
    first, second = ops.workspace(100, "cuda:0"), ops.workspace(100, "cuda:0")
    assert first.data_ptr() != second.data_ptr() and made == ["cuda:0"] * 2
    like = torch.zeros(1)
    a, b = ops._scratch(100, 0, 7, like), ops._scratch(100, 0, 7, like)
    assert a[0] != b[0]
    assert not ops._workspaces and not ops._q8_scratch
