"""Streams and graphs for the GPU tests, on the HIP runtime that the library loads."""
from __future__ import annotations

import ctypes as C

from bench import Hip


class Graphs:
    """A stream of its own; capture(fn) gives a graph of what fn(stream) enqueues, replay(graph) runs it and waits."""

    def __init__(self):
        self.hip = Hip()
        s = C.c_void_p()
        self.hip.ok(self.hip.lib.hipStreamCreateWithFlags(C.byref(s), 1), "hipStreamCreateWithFlags")
        self.stream = s.value

    def capture(self, fn):
        return self.hip.capture(self.stream, lambda: fn(self.stream))[0]

    def replay(self, *graphs):
        for g in graphs:
            self.hip.launch_graph(g, self.stream)
        self.hip.sync()

    def sync(self):
        self.hip.sync()
