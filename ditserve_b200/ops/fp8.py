"""8-bit activations: RMS norm with a quantised output, and the linear layer that reads it.

``rms_norm_quant(x, w, residual=r)`` adds the residual, normalises and leaves float8 e4m3 rows with
one fp32 scale each; ``linear_fp8`` multiplies such rows by weights that ``quantize_rows_fp8`` laid
out once, with the epilogues of ``linear``.  On CPU the same math runs in fp32 with PyTorch.  The
ops have no gradient.
"""
from __future__ import annotations

import torch

from ._ext import launch, status_word, use_kernels
from ._memory import shares_memory
from .gemm import _row_gate, gelu_tanh_ref

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0     # the largest finite float8 e4m3
SCALE_MIN = 1e-30    # scale of a row of zeros
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def empty_fp8(rows: int, cols: int, device=None) -> torch.Tensor:
    """Uninitialised e4m3 [rows, cols] whose rows start on 16 bytes, as ``linear_fp8`` reads them."""
    pitch = -(-cols // 16) * 16
    buf = torch.empty(rows, pitch, device=device, dtype=E4M3)
    return buf if pitch == cols else buf[:, :cols]


def quantize_rows_fp8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[rows, cols] -> (e4m3 [rows, cols], fp32 scale [rows]); a row is about ``q * scale``.

    Meant for weights, once at load; activations come from ``rms_norm_quant``."""
    if w.dim() != 2 or w.shape[1] == 0 or w.dtype not in _TYPES:
        raise ValueError("quantize_rows_fp8 takes a bf16, fp16 or fp32 matrix")
    f = w.float()
    scale = (f.abs().amax(dim=1) / E4M3_MAX).clamp_min(SCALE_MIN)
    q = empty_fp8(w.shape[0], w.shape[1], w.device)
    q.copy_((f / scale[:, None]).to(E4M3))
    return q, scale


def rms_norm_quant_reference(x, weight=None, residual=None, eps=1e-6):
    """fp32 PyTorch statement of the op (CPU path and test oracle): (q, scale, h or None)."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    scale = (y.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
    return (y / scale[..., None]).to(E4M3), scale, None if residual is None else h


def _rows_view(t: torch.Tensor, width: int, name: str) -> torch.Tensor:
    if t.dim() == 2:
        return t
    try:
        return t.view(-1, width)
    except RuntimeError as exc:
        raise ValueError(f"{name} must be viewable as rows of {width}") from exc


def _partial_overlap(out: torch.Tensor, src: torch.Tensor) -> bool:
    """Whether ``out`` shares memory with ``src`` other than element by element (both 2-D rows)."""
    same = out.data_ptr() == src.data_ptr() and out.element_size() == src.element_size() and out.shape == src.shape and \
        (out.shape[0] <= 1 or out.stride(0) == src.stride(0))
    return not same and shares_memory(out, src)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
                   eps: float = 1e-6, out: torch.Tensor | None = None, scale_out: torch.Tensor | None = None,
                   residual_out: torch.Tensor | None = None):
    """h = x + residual; y = h * rsqrt(mean(h^2) + eps) * weight; (q, scale) = e4m3 rows of y.

    x: [..., D] in bf16, fp16 or fp32, any row stride; weight [D] in the same type.  Returns
    (q, scale, h): q float8_e4m3fn [..., D] with rows on 16 bytes, scale fp32 [...] with
    y ~ q * scale[..., None], scale = max(max|y| / 448, 1e-30), and h in x's type (None without a
    residual).  The norm reads h as it is stored.  ``residual_out`` may be ``residual`` or ``x`` itself; the
    outputs share no memory with each other (columns of one buffer are apart).
    A NaN or an infinity in a row makes the row's scale and q NaN.  Squares are summed in fp32: rows whose
    sum(h^2) passes 3.4e38 are not represented (their q is zero)."""
    if x.is_cuda:
        got = launch("rms_norm_quant", x, weight, residual, eps, out, scale_out, residual_out)
        if got is not None:
            return got
    if x.dtype not in _TYPES:
        raise ValueError("rms_norm_quant takes bf16, fp16 or fp32")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("rms_norm_quant needs rows of at least one element")
    shape, d = x.shape, x.shape[-1]
    if weight is not None and (weight.shape != (d,) or weight.dtype != x.dtype):
        raise ValueError(f"weight must be [{d}] in x's type")
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise ValueError("residual must have x's shape and type")
    if residual_out is not None and (residual is None or residual_out.shape != shape or residual_out.dtype != x.dtype):
        raise ValueError("residual_out goes with a residual and has x's shape and type")
    if out is not None and (out.shape != shape or out.dtype != E4M3):
        raise ValueError("out must be float8_e4m3fn of x's shape")
    if scale_out is not None and (scale_out.shape != shape[:-1] or scale_out.dtype != torch.float32):
        raise ValueError("scale_out must be fp32 of x's shape without its last axis")
    outs = [t for t in (out, scale_out, residual_out) if t is not None]
    if any(shares_memory(a, b) for i, a in enumerate(outs) for b in outs[i + 1:]):
        raise ValueError("out, scale_out and residual_out must not share memory")
    if weight is not None and any(t is not None and shares_memory(t, weight) for t in (out, residual_out)):
        raise ValueError("out and residual_out must not share memory with weight")
    if not use_kernels(x, weight, residual, out, scale_out, residual_out):
        q, s, h = rms_norm_quant_reference(x, weight, residual, eps)
        q = q if out is None else out.copy_(q)
        s = s if scale_out is None else scale_out.copy_(s)
        h = h if residual_out is None else residual_out.copy_(h)
        return q, s, h
    # what the kernel does not take as it is: columns apart, outputs in other layouts
    x2, r2, h2 = x.reshape(-1, d), None, None
    x2 = x2 if x2.stride(1) == 1 or d == 1 else x2.contiguous()
    q2 = empty_fp8(x2.shape[0], d, x.device) if out is None else _rows_view(out, d, "out")
    s1 = torch.empty(x2.shape[0], device=x.device, dtype=torch.float32)
    if out is not None and any(t is not None and _partial_overlap(q2, t.reshape(-1, d)) for t in (x, residual, residual_out)):
        raise ValueError("out overlaps the other tensors")
    if residual is not None:
        r2 = residual.reshape(-1, d)
        r2 = r2 if r2.stride(1) == 1 or d == 1 else r2.contiguous()
        h2 = torch.empty(x2.shape[0], d, device=x.device, dtype=x.dtype) if residual_out is None else \
            _rows_view(residual_out, d, "residual_out")
        if residual_out is not None and (_partial_overlap(h2, x2) or _partial_overlap(h2, r2)):
            raise ValueError("residual_out overlaps its inputs without being one of them")
    weight = weight if weight is None else weight.contiguous()
    if launch("rms_norm_quant", x2, weight, r2, eps, q2, s1, h2) is None:
        raise ValueError("rms_norm_quant needs its tensors on one CUDA device and outputs with packed, separate rows")
    scale = s1.view(shape[:-1]) if scale_out is None else scale_out.copy_(s1.view(shape[:-1]))
    return (q2.view(shape) if out is None else out, scale,
            None if residual is None else (h2.view(shape) if residual_out is None else residual_out))


def linear_fp8_reference(xq, x_scale, wq, w_scale, b=None, act=None, residual=None, gate=None, rows_per_batch=None,
                         row_batch=None, out_dtype=torch.bfloat16):
    """fp32 PyTorch statement of the op (CPU path and test oracle)."""
    shape = xq.shape
    y = xq.reshape(-1, shape[-1]).float() @ wq.float().t()
    y = y * x_scale.reshape(-1, 1) * w_scale
    if b is not None:
        y = y + b.float()
    if act == "gelu":
        y = gelu_tanh_ref(y)
    if gate is not None:
        y = y * _row_gate(gate, y.shape[0], rows_per_batch, row_batch)
    if residual is not None:
        y = y + residual.reshape(y.shape).float()
    return y.to(out_dtype).reshape(*shape[:-1], wq.shape[0])


def _aligned_rows(q: torch.Tensor) -> torch.Tensor:
    """``q`` itself if its rows start on 16 bytes, else a copy whose rows do."""
    ok = (q.shape[1] == 1 or q.stride(1) == 1) and q.data_ptr() % 16 == 0 and \
        (q.shape[0] <= 1 or (q.stride(0) % 16 == 0 and q.stride(0) >= q.shape[1]))
    return q if ok else empty_fp8(q.shape[0], q.shape[1], q.device).copy_(q)


def linear_fp8(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
               b: torch.Tensor | None = None, *, act: str | None = None, residual: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, rows_per_batch: int | None = None,
               row_batch: torch.Tensor | None = None, out: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y = epilogue(x_scale[m] * w_scale[n] * sum_k xq[m, k] wq[n, k] + b[n]), epilogues as in ``linear``.

    xq: float8_e4m3fn [..., K] with fp32 x_scale [...]; wq float8_e4m3fn [N, K] with fp32 w_scale [N]
    (``quantize_rows_fp8``).  Any M and N up to 2^30, K up to 2^28; rows that do not start on 16 bytes (K not a multiple
    of 16 in a packed matrix) are copied first on every call, which ``empty_fp8`` avoids.  The result, b and residual share
    ``out_dtype`` (bf16, fp16 or fp32; ``out`` decides if given).  ``out`` may be ``residual`` itself, but shares no memory
    with what else is read (columns of one buffer are apart).
    gate is fp32 [N] or [B, N] and needs a residual; row m takes gate row m // rows_per_batch, or
    row_batch[m] (entries outside [0, B) take the nearest row)."""
    if xq.is_cuda and act in (None, "gelu"):
        y = launch("linear_fp8", xq, x_scale, wq, w_scale, b, act is not None, residual, gate, rows_per_batch, row_batch,
                   out, out_dtype)
        if y is not None:
            return y
    if xq.dtype != E4M3 or wq.dtype != E4M3:
        raise ValueError("xq and wq must be float8_e4m3fn")
    if xq.dim() < 1 or wq.dim() != 2 or xq.shape[-1] != wq.shape[1] or wq.shape[1] == 0:
        raise ValueError("xq [..., K] and wq [N, K] must share K >= 1")
    lead, K, N = xq.shape[:-1], wq.shape[1], wq.shape[0]
    if K > 1 << 28 or N > 1 << 30 or xq.numel() // K > 1 << 30:
        raise ValueError("linear_fp8 takes up to 2^28 values and 2^30 rows and channels")
    if x_scale.dtype != torch.float32 or x_scale.shape != lead:
        raise ValueError("x_scale must be fp32 of xq's shape without its last axis")
    if w_scale.dtype != torch.float32 or w_scale.shape != (N,):
        raise ValueError(f"w_scale must be fp32 [{N}]")
    if act not in (None, "gelu"):
        raise ValueError(f"unsupported activation {act!r}")
    if act is not None and residual is not None:
        raise ValueError("activation and residual epilogues are exclusive")
    if out is not None:
        out_dtype = out.dtype
        if out.shape != (*lead, N):
            raise ValueError(f"out must be {(*lead, N)}")
    if out_dtype not in _TYPES:
        raise ValueError("the result is bf16, fp16 or fp32")
    if b is not None and (b.shape != (N,) or b.dtype != out_dtype):
        raise ValueError(f"b must be [{N}] in the result's type")
    if residual is not None and (residual.shape != (*lead, N) or residual.dtype != out_dtype):
        raise ValueError("residual must have the result's shape and type")
    M = x_scale.numel()
    if gate is not None:
        if residual is None:
            raise ValueError("a gate needs a residual")
        if gate.dim() == 1:
            gate = gate.unsqueeze(0)
        if gate.dtype != torch.float32 or gate.dim() != 2 or gate.shape[0] == 0 or gate.shape[1] != N:
            raise ValueError(f"gate must be fp32 [{N}] or [B, {N}]")
        if row_batch is not None:
            if row_batch.dtype != torch.int32 or row_batch.shape != (M,):
                raise ValueError(f"row_batch must be int32 [{M}]")
        elif rows_per_batch is not None and (rows_per_batch < 1 or -(-M // rows_per_batch) > gate.shape[0]):
            raise ValueError("rows_per_batch must be positive and gate have a row for every batch")
    if out is not None and any(t is not None and shares_memory(out, t) for t in (
            x_scale, w_scale, b, gate, row_batch if gate is not None else None)):
        raise ValueError("out must not share memory with scales, b, gate or row_batch")
    if not use_kernels(xq, wq, x_scale, w_scale, b, residual, gate, out):
        if row_batch is not None and gate is not None:
            row_batch = row_batch.clamp(0, gate.shape[0] - 1)
        y = linear_fp8_reference(xq, x_scale, wq, w_scale, b, act, residual, gate, rows_per_batch, row_batch, out_dtype)
        return y if out is None else out.copy_(y)
    # what the kernel does not take as it is: rows off 16 bytes, columns apart, the first call on a device
    status_word(xq.device)
    y2 = torch.empty(M, N, device=xq.device, dtype=out_dtype) if out is None else _rows_view(out, N, "out")
    r2 = None
    if residual is not None:
        r2 = residual.reshape(-1, N)
        r2 = r2 if r2.stride(1) == 1 or N == 1 else r2.contiguous()
        if out is not None and _partial_overlap(y2, r2):
            raise ValueError("out overlaps the residual without being it")
    x2, w2 = _aligned_rows(xq.reshape(-1, K)), _aligned_rows(wq)
    if out is not None and (_partial_overlap(y2, x2) or _partial_overlap(y2, w2)):
        raise ValueError("out overlaps the operands")
    got = launch("linear_fp8", x2, x_scale.reshape(-1).contiguous(), w2,
                 w_scale.contiguous(), b if b is None else b.contiguous(), act is not None, r2,
                 gate if gate is None or gate.stride(1) == 1 else gate.contiguous(), rows_per_batch,
                 row_batch if row_batch is None else row_batch.contiguous(), y2, out_dtype)
    if got is None:
        raise ValueError("linear_fp8 needs its tensors on one CUDA device and out with packed, separate rows")
    return y2.view(*lead, N) if out is None else out
