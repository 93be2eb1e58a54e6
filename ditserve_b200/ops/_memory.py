"""Whether tensors share bytes, for the checks of outputs against what a call reads or writes besides."""
from __future__ import annotations

import math

import torch


def _runs(t: torch.Tensor):
    """(first byte, one behind the last, bytes of a run, runs, pitch); one run over the whole span where the
    tensor is not equally spaced runs."""
    e, lo = t.element_size(), t.data_ptr()
    dims = sorted((st * e, n) for n, st in zip(t.shape, t.stride()) if n > 1 and st)
    hi = lo + e + sum(st * (n - 1) for st, n in dims)
    run, i = e, 0
    while i < len(dims) and dims[i][0] == run:
        run *= dims[i][1]
        i += 1
    if i == len(dims):
        return lo, hi, hi - lo, 1, 0
    pitch, count = dims[i]
    for st, n in dims[i + 1:]:
        if st != pitch * count:
            return lo, hi, hi - lo, 1, 0
        count *= n
    return (lo, hi, run, count, pitch) if run <= pitch else (lo, hi, hi - lo, 1, 0)


def shares_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether ``a`` and ``b`` have a byte in common.  Columns of one buffer are told apart; for layouts that are
    not equally spaced rows the answer is whether their spans meet."""
    if not a.numel() or not b.numel() or a.device != b.device:
        return False
    a0, a1, run_a, n_a, pitch_a = _runs(a)
    b0, b1, run_b, n_b, pitch_b = _runs(b)
    if a1 <= b0 or b1 <= a0:
        return False
    pitch = math.gcd(pitch_a, pitch_b)  # all runs of either start in one place of it
    if not pitch:
        return True
    d = (a0 - b0) % pitch
    return d < run_b or d + run_a > pitch
