"""Whether tensors share bytes, for the checks of outputs against what a call reads or writes besides."""
from __future__ import annotations

import math

import torch


def _runs(t: torch.Tensor):
    """(first byte, one behind the last, bytes of a run, a pitch that divides the runs' distances); one run over the
    whole span, and a pitch of 0, where runs do not fit into such a pitch."""
    e, lo = t.element_size(), t.data_ptr()
    dims = sorted((st * e, n) for n, st in zip(t.shape, t.stride()) if n > 1 and st)
    hi = lo + e + sum(st * (n - 1) for st, n in dims)
    run, i = e, 0
    while i < len(dims) and dims[i][0] == run:
        run *= dims[i][1]
        i += 1
    if i == len(dims):
        return lo, hi, hi - lo, 0
    pitch = math.gcd(*(st for st, _ in dims[i:]))  # every run starts in one place of it
    return (lo, hi, run, pitch) if run <= pitch else (lo, hi, hi - lo, 0)


def shares_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``a`` and ``b`` have a byte in common.  Columns of one buffer are told apart; for layouts
    without rows in columns the answer is whether their spans meet."""
    if not a.numel() or not b.numel() or a.device != b.device:
        return False
    a0, a1, run_a, pitch_a = _runs(a)
    b0, b1, run_b, pitch_b = _runs(b)
    if a1 <= b0 or b1 <= a0:
        return False
    pitch = math.gcd(pitch_a, pitch_b)  # all runs of either start in one place of it
    if not pitch:
        return True
    d = (a0 - b0) % pitch
    return d < run_b or d + run_a > pitch
