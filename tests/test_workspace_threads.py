"""The table of scratch buffers under several host threads."""
import contextlib
import threading
import types

import torch

from mlx_b200 import ops


def test_threads_that_need_the_first_buffer_at_once_get_the_same(monkeypatch):
    """Whoever comes while a buffer is being made waits for it: with one each, the native form could keep the address of the one that
    the table dropped."""
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: types.SimpleNamespace(cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    told, made, zeros = [], threading.Event(), torch.zeros

    def slow_zeros(*a, **kw):
        made.wait(0.2)   # until another thread asks for a buffer too, or for a while
        made.set()
        return zeros(*a, **kw)

    monkeypatch.setattr(torch, "zeros", slow_zeros)
    monkeypatch.setattr(ops, "_front", types.SimpleNamespace(scratch=lambda *a: told.append(a[3])))
    spaces, dev, got = ops._Workspaces(), torch.device("cpu:0"), []
    threads = [threading.Thread(target=lambda: got.append(spaces.get(dev, 1000, "qmm"))) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len({b.data_ptr() for b in got}) == 1 and told == [got[0].data_ptr()]
    assert [b.data_ptr() for _, b in spaces.all()] == told
