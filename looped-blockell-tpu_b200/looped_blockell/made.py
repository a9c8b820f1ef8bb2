"""Device tensors that a cache hands out, on whatever stream asks for them."""

from __future__ import annotations

import torch

_capturing = torch.cuda.is_current_stream_capturing
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def capturing(t: torch.Tensor) -> bool:
    """Whether work on ``t`` is being captured: what is made then holds nothing until a replay."""
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class Made:
    """The tensors of one cache entry, made by work on the current stream (not
    while it is captured).  ``use`` before each further use: another stream
    waits for that work, and the memory is not reused before that stream's own.
    In a capture it does neither: a graph cannot wait for work outside it, so a
    capture begins after what was made before it (``torch.cuda.graph``
    synchronises first).  Its replays read the memory again: what a graph has
    ``captured`` must outlive the entry."""

    __slots__ = ("tensors", "index", "stream", "event", "captured")

    def __init__(self, *tensors: torch.Tensor):
        self.tensors = tensors if tensors[0].is_cuda else ()
        self.captured = False
        if self.tensors:
            s = torch.cuda.current_stream(tensors[0].device)
            self.index, self.stream, self.event = s.device_index, s.cuda_stream, s.record_event()

    def use(self) -> None:
        if not self.tensors:
            return
        if _capturing():
            self.captured = True
        elif _raw_stream(self.index) != self.stream:
            self._order()

    def _order(self) -> None:
        s = torch.cuda.current_stream(self.index)
        s.wait_event(self.event)
        for t in self.tensors:
            t.record_stream(s)
