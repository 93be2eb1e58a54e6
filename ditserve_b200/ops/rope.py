"""Rotary positions with several axes (time, height, width) for image and video tokens.

``rope_axes`` rotates queries and keys by positions given for every token and axis, so ragged and
packed token lists need no table per grid (``rmsnorm_rope_`` reads such tables).  On CPU the same
math runs in PyTorch.  The op has no gradient of its own; ``inverse=True`` is its transpose.
"""
from __future__ import annotations

import functools

import torch

from ._ext import ext, launch, use_kernels
from ._memory import shares_memory
from .fp8 import _partial_overlap, _rows_view

_POSITIONS = (torch.int64, torch.int32, torch.float32, torch.float64)
MAX_AXES, MAX_ROTATED = 4, 512


def grid_positions(grid, device=None) -> torch.Tensor:
    """int64 [t * h * w, 3] (or any number of axes): the raster positions of a token grid."""
    axes = torch.meshgrid(*[torch.arange(n, device=device) for n in grid], indexing="ij")
    return torch.stack(axes, -1).reshape(-1, len(grid))


def rope_axes_reference(x, positions, dims, head_dim, theta, layout="interleaved", inverse=False):
    """PyTorch statement of the op for one tensor [rows, heads * head_dim]: fp64 angles, fp32 rotation."""
    axis = torch.cat([torch.full((d // 2,), i) for i, d in enumerate(dims)]).to(x.device)
    freq = torch.cat([float(t) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for d, t in zip(dims, theta)])
    angle = positions.double()[:, axis] * freq.to(x.device)
    angle = angle.repeat(x.shape[0] // max(positions.shape[0], 1), 1)[:, None]
    cos, sin = angle.cos().float(), angle.sin().float() * (-1 if inverse else 1)
    n = sum(dims) // 2
    f = x.float().reshape(x.shape[0], -1, head_dim)
    y = f.clone()
    a, b = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y[..., a] = f[..., a] * cos - f[..., b] * sin
    y[..., b] = f[..., a] * sin + f[..., b] * cos
    return y.reshape(x.shape).to(x.dtype)


@functools.lru_cache(maxsize=64)
def _plan(dims: tuple, theta):
    """The frequencies of a set of axes, or None where dims or theta are wrong (the caller says how)."""
    thetas = [float(theta)] * len(dims) if isinstance(theta, (int, float)) else list(theta)
    return ext().rope_plan(list(dims), thetas)


def rope_axes(x: torch.Tensor, positions: torch.Tensor, dims, *, k: torch.Tensor | None = None, head_dim: int = 128,
              theta=10000.0, layout: str = "interleaved", inverse: bool = False, out: torch.Tensor | None = None,
              k_out: torch.Tensor | None = None):
    """Rotates x (and k) [..., heads * head_dim] by each token's positions; returns the result or (x', k').

    positions: [P, axes] (or [P] for one axis), int64, int32, fp32 or fp64, any strides; row r takes
    position r % P, so a batch may share them.  dims: rotated elements of each axis, even, at most
    head_dim together; elements behind them pass through.  Pair j of an axis of d elements turns by
    position * theta^(-2j / d); theta is one number or one for each axis.  layout "interleaved" pairs
    elements (2i, 2i + 1), "half" pairs (i, i + sum(dims) / 2).  inverse turns the other way.  x and k
    (bf16, fp16 or fp32) may differ in heads.  out / k_out may be x / k themselves; they share no memory with
    what else is read or written (columns of one buffer are apart)."""
    if x.is_cuda and layout in ("interleaved", "half"):
        # by value: a tensor among them would be told apart by its identity
        plan = _plan(tuple(map(int, dims)),
                     theta if isinstance(theta, (int, float)) else tuple(map(float, theta)))
        if plan is not None:
            got = launch("rope_axes", x, k, positions, plan, head_dim, layout == "half", inverse, out, k_out)
            if got is not None:
                return got
    dims = tuple(int(d) for d in dims)
    if not 1 <= len(dims) <= MAX_AXES or any(d <= 0 or d % 2 for d in dims):
        raise ValueError(f"dims must be 1 to {MAX_AXES} positive even numbers")
    if head_dim < 1 or sum(dims) > min(head_dim, MAX_ROTATED):
        raise ValueError(f"dims must sum to at most head_dim and {MAX_ROTATED}")
    theta = (float(theta),) * len(dims) if isinstance(theta, (int, float)) else tuple(float(t) for t in theta)
    if len(theta) != len(dims) or any(not 0 < t < float("inf") for t in theta):
        raise ValueError("theta must be positive, one number or one for each axis")
    if layout not in ("interleaved", "half"):
        raise ValueError(f"unknown layout {layout!r}")
    if positions.dim() == 1 and len(dims) == 1:
        positions = positions.unsqueeze(1)
    if positions.dim() != 2 or positions.shape[1] != len(dims) or positions.dtype not in _POSITIONS:
        raise ValueError(f"positions must be int64, int32, fp32 or fp64 [P, {len(dims)}]")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("rope_axes takes bf16, fp16 or fp32")
    if x.dim() < 2 or x.shape[-1] == 0 or x.shape[-1] % head_dim:
        raise ValueError("x must be [..., heads * head_dim]")
    rows = x.numel() // x.shape[-1]
    if rows and (positions.shape[0] == 0 or rows % positions.shape[0]):
        raise ValueError("the tokens must be a multiple of the positions")
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype):
        raise ValueError("out must have x's shape and type")
    if k is None:
        if k_out is not None:
            raise ValueError("k_out goes with k")
    else:
        if k.dtype != x.dtype or k.dim() < 2 or k.shape[-1] == 0 or k.shape[-1] % head_dim or k.numel() // k.shape[-1] != rows:
            raise ValueError("k must be [..., heads * head_dim] with x's tokens and type")
        if k_out is not None and (k_out.shape != k.shape or k_out.dtype != k.dtype):
            raise ValueError("k_out must have k's shape and type")
    if out is not None and k_out is not None and shares_memory(out, k_out):
        raise ValueError("the outputs of x and k must be apart")
    if any(o is not None and shares_memory(o, positions) for o in (out, k_out)):
        raise ValueError("out and k_out must not share memory with positions")
    if not use_kernels(x, positions, k, out, k_out):
        # both are rotated before either is stored: out may lie on k
        got = [rope_axes_reference(t.reshape(-1, t.shape[-1]), positions, dims, head_dim, theta, layout, inverse)
               .reshape(t.shape) for t in (x, k) if t is not None]
        got = [r if o is None else o.copy_(r) for r, o in zip(got, (out, k_out))]
        return got[0] if k is None else tuple(got)
    # what the kernel does not take as it is: columns apart, several outputs to tell apart
    t2, o2, w = [], [], [x.shape[-1], 0 if k is None else k.shape[-1]]
    for i, (t, o) in enumerate(((x, out), (k, k_out))):
        if t is None:
            t2.append(None), o2.append(None)
            continue
        t2.append(t.reshape(-1, w[i]))
        if t2[i].stride(1) != 1 and w[i] > 1:
            t2[i] = t2[i].contiguous()
        o2.append(torch.empty(rows, w[i], device=x.device, dtype=x.dtype) if o is None else _rows_view(o, w[i], "out"))
    if rows and (out is not None or k_out is not None):
        if any(_partial_overlap(a, b) for a in o2 if a is not None for b in t2 if b is not None):
            raise ValueError("an output overlaps an input without being it")
        if k is not None and (o2[0].data_ptr() == o2[1].data_ptr() or _partial_overlap(o2[0], o2[1])
                              or o2[0].data_ptr() == t2[1].data_ptr() or o2[1].data_ptr() == t2[0].data_ptr()):
            raise ValueError("the outputs of x and k must be apart")
    if launch("rope_axes", t2[0], t2[1], positions, _plan(dims, theta), head_dim, layout == "half", inverse, o2[0],
              o2[1]) is None:
        raise ValueError("rope_axes needs its tensors on one CUDA device and outputs with packed, separate rows")
    x2 = o2[0].view(x.shape) if out is None else out
    return x2 if k is None else (x2, o2[1].view(k.shape) if k_out is None else k_out)
