"""Greedy and temperature sampling over the step's logits.

Greedy is the reference's rule: the smallest index attaining the maximum
(imparo-cpu/src/ops.rs:628-640).  The reference samples with nothing else — its
temperature argument is ignored (imparo-server/src/main.rs:3383-3390).  Temperature
sampling here: p = softmax(logits / T) in 32-bit, one uniform number u per (seed, step)
from a counter-based generator, and the pick is the first index whose running sum of p
in vocabulary order exceeds u * sum(p).  T == 0 is greedy.

A request may also filter its tokens: top-k, then top-p of what that leaves, then min-p (ops.sample_filtered).  Its
pick is made in sums that are exact for all practical purposes; requests without a filter are picked as above, whatever
the others of the step ask for.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from ..kernels import ops

_MASK = (1 << 64) - 1


def uniform_for(seed: int, step: int) -> float:
    """u in [0, 1) with 24 bits, a pure function of (seed, step): splitmix64 of
    seed * 0x9E3779B97F4A7C15 + step."""
    z = ((int(seed) & _MASK) * 0x9E3779B97F4A7C15 + (int(step) & _MASK) + 0x9E3779B97F4A7C15) & _MASK
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _MASK
    z ^= z >> 31
    return (z >> 40) / float(1 << 24)


class PendingSample:
    """Ids sampled on the device whose copy to the host is under way.  dev_ids can feed the
    next step on the device at once; result() waits for the copy and returns the ids."""

    def __init__(self, dev_ids: torch.Tensor, host_ids: torch.Tensor, event: torch.cuda.Event):
        self.dev_ids, self._host, self._event = dev_ids, host_ids, event

    def result(self) -> List[int]:
        self._event.synchronize()
        return self._host.tolist()


class Sampler:
    RING = 3        # a step's ids stay valid while the next two steps sample

    def __init__(self, device, max_rows: int = 1024):
        self.device = device
        self._cap = 0
        self._turn = 0
        self._grow(max_rows)

    def _grow(self, n: int) -> None:
        if n <= self._cap:
            return
        self._cap = n
        # per row: temperature, uniform number; top_p, min_p, and as whole numbers top_k and whether the row filters
        self._host_in = [torch.empty((6, n), dtype=torch.float32, pin_memory=True) for _ in range(self.RING)]
        self._dev_in = torch.empty((6, n), dtype=torch.float32, device=self.device)
        self._dev_filtered = torch.empty(n, dtype=torch.int32, device=self.device)
        self._dev_outs = [torch.empty(n, dtype=torch.int32, device=self.device) for _ in range(self.RING)]
        self._host_outs = [torch.empty(n, dtype=torch.int32, pin_memory=True) for _ in range(self.RING)]

    def sample(self, logits: torch.Tensor, temperatures: Optional[Sequence[float]] = None,
               seeds: Optional[Sequence[int]] = None, steps: Optional[Sequence[int]] = None,
               top_ks: Optional[Sequence[int]] = None, top_ps: Optional[Sequence[float]] = None,
               min_ps: Optional[Sequence[float]] = None) -> List[int]:
        """One token id per row of logits.  temperatures None or all 0: greedy.  Row r with
        temperature > 0 uses uniform_for(seeds[r], steps[r]).  top_ks, top_ps, min_ps: a filter per row each, or None
        (0 or less, 1 or more, 0 or less: that row has none).  Reads the ids back (this is
        the step's device-to-host copy) and returns them as a list."""
        return self.sample_async(logits, temperatures, seeds, steps, top_ks, top_ps, min_ps).result()

    def sample_async(self, logits: torch.Tensor, temperatures: Optional[Sequence[float]] = None,
                     seeds: Optional[Sequence[int]] = None, steps: Optional[Sequence[int]] = None,
                     top_ks: Optional[Sequence[int]] = None, top_ps: Optional[Sequence[float]] = None,
                     min_ps: Optional[Sequence[float]] = None) -> PendingSample:
        """Like sample(), without waiting: the kernels and the device-to-host copy are queued."""
        n = logits.shape[0]
        self._grow(n)
        self._turn = (self._turn + 1) % self.RING
        out = self._dev_outs[self._turn][:n]
        if temperatures is None or not any(t > 0 for t in temperatures):
            ops.sample_rows(logits, None, None, out)
        else:
            h = self._host_in[self._turn]
            hn = h.numpy()                      # the same pinned memory: element writes without tensor indexing
            filtered = 0
            if top_ks is not None or top_ps is not None or min_ps is not None:
                whole = hn.view(np.int32)
                for r in range(n):
                    k = min(int(top_ks[r]), 1 << 30) if top_ks is not None else 0
                    p = float(top_ps[r]) if top_ps is not None else 1.0
                    m = float(min_ps[r]) if min_ps is not None else 0.0
                    hn[2, r], hn[3, r], whole[4, r] = p, m, max(k, 0)
                    whole[5, r] = filters = temperatures[r] > 0 and (k > 0 or p < 1 or m > 0)
                    filtered += filters
            for r in range(n):
                t = float(temperatures[r])
                hn[0, r] = t
                hn[1, r] = uniform_for(seeds[r], steps[r]) if t > 0 else 0.0
            dev = self._dev_in[:6 if filtered else 2, :n]
            dev.copy_(h[:6 if filtered else 2, :n], non_blocking=True)
            if filtered < n:
                ops.sample_rows(logits, dev[0], dev[1], out)
            if filtered:
                picked = out if filtered == n else self._dev_filtered[:n]
                ops.sample_filtered(logits, dev[0], dev[1], picked, top_k=dev[4].view(torch.int32), top_p=dev[2], min_p=dev[3])
                if picked is not out:
                    torch.where(dev[5].view(torch.int32) != 0, picked, out, out=out)
        host = self._host_outs[self._turn][:n]
        host.copy_(out, non_blocking=True)
        ev = torch.cuda.Event()
        ev.record()
        return PendingSample(out, host, ev)
