"""The serving operators' Python side without a GPU."""

from __future__ import annotations

import threading
import time

from so101_smolvla_edge_b200 import _lib as L
from so101_smolvla_edge_b200 import ops


def test_threads_share_one_workspace(monkeypatch):
    """Two threads whose first calls on a stream meet: the arrays that the native side was given are the ones kept."""

    class Fake:
        nbytes = 0

        def __init__(self, *_, **__):
            time.sleep(0.05)  # allocating lets the other thread run
            self.partials = self.tickets = self

        def data_ptr(self):
            return id(self)

        def numel(self):
            return 0

    registered = []

    class Calls:
        @staticmethod
        def add_workspace(device, stream, partials, *_):
            time.sleep(0.05 if not registered else 0.0)
            registered.append(partials)

    monkeypatch.setattr(ops, "Workspace", Fake)
    monkeypatch.setattr(ops, "_PAGES_WS", {})
    monkeypatch.setattr(L, "calls", lambda: Calls)
    got = []
    threads = [threading.Thread(target=lambda: got.append(ops.pages_workspace(0, 7))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert registered == [id(ops._PAGES_WS[0, 7])]
    assert len({id(w) for w in got}) == 1
