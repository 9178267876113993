"""Device-side error counts read without stalling the host.

Some operators count bad inputs on the device (the fused CE's out-of-range
labels, the splice's placeholder count and out-of-range ids).  Reading such a
count at once would synchronise the host with the GPU on every call, so each
call copies its counts to pinned host memory without blocking, records an
event, and the counts are judged once the copy has landed: at the operator's
next call, or when the caller asks (``check(block=True)``, e.g. at the end
of a training or evaluation loop).  An operator may also write them there itself
(``landing`` and ``landed_on``): a copy takes 8 us of the stream.  Inside HIP graph capture neither the copy
nor an event query of earlier work is allowed, so captured calls are not
tracked.
"""

from __future__ import annotations

import threading
from typing import Callable

import torch


class DeferredChecks:
    """Pending device counts of one operator, each with the function that
    judges them (raises on bad values)."""

    def __init__(self) -> None:
        self._pending: list = []
        self._lock = threading.Lock()

    def add(self, counts: torch.Tensor, judge: Callable[[list], None]) -> None:
        """Tracks ``counts`` (a small int64 device tensor); ``judge`` gets its
        values as a Python list once they have landed."""
        if torch.cuda.is_current_stream_capturing():
            return
        self.check()
        host = torch.empty(counts.shape, dtype=counts.dtype, pin_memory=True)
        host.copy_(counts, non_blocking=True)
        call = self._call(counts.device, host, judge)
        with self._lock:
            self._pending.append(call)

    def landing(self, n: int) -> torch.Tensor | None:
        """Pinned memory for ``n`` counts of a call that writes them by itself
        (None while a graph is captured); ``landed_on`` follows the call."""
        if torch.cuda.is_current_stream_capturing():
            return None
        return torch.empty(n, dtype=torch.int64, device="cpu", pin_memory=True)

    def landed_on(self, device: torch.device, host: torch.Tensor, judge: Callable[[list], None]) -> None:
        """Tracks the counts that the work now on ``device``'s current stream
        leaves in ``host``, which is held until it has."""
        call = self._call(device, host, judge)
        try:
            self.check()
        finally:
            with self._lock:
                self._pending.append(call)

    def hold(self, device: torch.device, host: torch.Tensor) -> None:
        """Keeps ``host`` as ``landed_on`` does, for a call that failed: it may
        have been launched, and what it leaves there is not judged."""
        with self._lock:
            self._pending.append(self._call(device, host, lambda counts: None))

    @staticmethod
    def _call(device: torch.device, host: torch.Tensor, judge: Callable[[list], None]) -> tuple:
        ev = torch.cuda.Event()
        stream = torch.cuda.current_stream(device)
        ev.record(stream)
        return ev, (device, stream.cuda_stream), host, judge

    def check(self, block: bool = False) -> None:
        """Judges every tracked call whose counts have landed (all of them when
        ``block``); the first bad one raises, and each call is judged once."""
        landed = []
        behind = set()  # streams with a call that has not landed: later ones there have not either, and are not asked
        with self._lock:
            keep = []
            for call in self._pending:
                ev, where, host, judge = call
                if block:
                    ev.synchronize()
                if where not in behind and ev.query():
                    landed.append((host, judge))
                else:
                    behind.add(where)
                    keep.append(call)
            self._pending[:] = keep
        for host, judge in landed:
            judge(host.reshape(-1).tolist())

    def __len__(self) -> int:
        with self._lock:
            return len(self._pending)
