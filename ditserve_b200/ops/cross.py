"""Cross attention: queries of one length, an encoder's states of another, padded and masked.

``attention`` takes dense batches or packed lists; ``cross_attention`` takes padded batches as text
encoders leave them: every prompt in its own row of slots with a valid length or a key mask,
single queries (pooled tokens) to whole videos of them, shared key heads, bf16 and fp16.  On CPU the
same math runs in fp32 with PyTorch.  The op has no gradient.
"""
from __future__ import annotations

import math

import torch

from ._ext import launch, status_word, use_kernels
from ._memory import shares_memory

# fp32's smallest number; its largest over log2(e), which the exponentials' base takes in
SCALE_MIN, SCALE_MAX = 2.0 ** -149, torch.finfo(torch.float32).max / math.log2(math.e)


def cross_attention_reference(q, k, v, heads, heads_kv=None, kv_lens=None, key_mask=None, scale=None, return_lse=False):
    """fp32 PyTorch statement of the op for [B, S, heads * head_dim] tensors (CPU path and test oracle)."""
    heads_kv = heads_kv or heads
    B, Sq, width = q.shape
    Sk, d = k.shape[1], width // heads
    scale = scale if scale is not None else 1.0 / math.sqrt(d)
    allowed = torch.ones(B, Sk, dtype=torch.bool, device=q.device)
    if kv_lens is not None:
        allowed &= torch.arange(Sk, device=q.device) < kv_lens.to(q.device)[:, None]
    if key_mask is not None:
        allowed &= key_mask
    qh = q.float().reshape(B, Sq, heads, d).transpose(1, 2)
    kh = k.float().reshape(B, Sk, heads_kv, d).transpose(1, 2).repeat_interleave(heads // heads_kv, dim=1)
    vh = torch.where(allowed[..., None], v.float(), torch.zeros((), device=q.device))
    vh = vh.reshape(B, Sk, heads_kv, d).transpose(1, 2).repeat_interleave(heads // heads_kv, dim=1)
    s = (qh @ kh.transpose(-1, -2) * scale).masked_fill(~allowed[:, None, None], -math.inf)
    lse = torch.logsumexp(s, dim=-1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    o = (p @ vh).transpose(1, 2).reshape(B, Sq, width).to(q.dtype)
    return (o, lse) if return_lse else o


def _shares_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the spans of two tensors meet (columns of one buffer count as meeting)."""
    if not a.numel() or not b.numel() or a.device != b.device:
        return False

    def span(t):
        n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + n * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _meets_itself(t: torch.Tensor) -> bool:
    """Whether elements of ``t`` may lie on one another: axes that are not nested in one another count as that."""
    extent = 1
    for stride, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if stride < extent:
            return True
        extent += stride * (n - 1)
    return False


def _strided(t: torch.Tensor) -> torch.Tensor:
    ok = t.stride(2) == 1 and t.stride(1) % 8 == 0 and (t.stride(1) > 0 or t.shape[1] == 1) and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, heads: int, *, heads_kv: int | None = None,
                    kv_lens: torch.Tensor | None = None, key_mask: torch.Tensor | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scale * q k^T) v over the keys that are left of each batch entry.

    q [B, Sq, heads * head_dim], k and v [B, Sk, heads_kv * head_dim] in bf16 or fp16, head_dim 64 or
    128 (2-D tensors: one batch entry); head h reads key head h // (heads / heads_kv); at most 65535
    batch entries and key heads.  kv_lens: int32
    or int64 [B], the first kv_lens[b] keys are valid (held to 0 .. Sk); key_mask: bool [B, Sk], False
    keys are left out; both may be given.  What left-out slots of k and v hold does not matter, NaN and
    infinities included.  A query with no key left gets zeros and an lse of -inf.  scale is positive, 2^-149 to
    2.3e38, 1 / sqrt(head_dim) by default.  Any batch and row strides of at least 16 bytes' alignment are read in
    place, others copied first; a context may be shared through a batch stride of 0 (``expand``).
    Returns out [B, Sq, heads * head_dim], with return_lse also the fp32 natural-log sums [B, heads, Sq]."""
    heads_kv = heads if heads_kv is None else heads_kv
    if q.is_cuda:
        got = launch("cross_attention", q, k, v, heads, heads_kv, kv_lens, key_mask, scale, out, return_lse)
        if got is not None:
            return got
    if q.dim() == 2:
        if k.dim() != 2 or v.dim() != 2 or (out is not None and out.dim() != 2):
            raise ValueError("q, k, v and out must agree in dimensions")
        got = cross_attention(q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0), heads, heads_kv=heads_kv, kv_lens=kv_lens,
                              key_mask=key_mask, scale=scale, out=None if out is None else out.unsqueeze(0),
                              return_lse=return_lse)
        return (got[0][0], got[1][0]) if return_lse else got[0]
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [B, S, heads * head_dim]")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must be bf16 or fp16, all the same")
    if heads < 1 or heads_kv < 1 or heads % heads_kv:
        raise ValueError("heads must be a multiple of heads_kv")
    if q.shape[0] > 65535 or heads_kv > 65535:
        raise ValueError("at most 65535 batch entries and key heads")
    B, Sq, width = q.shape
    Sk, d = k.shape[1], width // heads
    if width % heads or d not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    if k.shape != (B, Sk, heads_kv * d) or v.shape != k.shape:
        raise ValueError(f"k and v must be [{B}, Sk, {heads_kv * d}]")
    if kv_lens is not None and (kv_lens.shape != (B,) or kv_lens.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"kv_lens must be int32 or int64 [{B}]")
    if key_mask is not None and (key_mask.shape != (B, Sk) or key_mask.dtype != torch.bool):
        raise ValueError(f"key_mask must be bool [{B}, {Sk}]")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not SCALE_MIN <= scale <= SCALE_MAX:
        raise ValueError("scale must be positive and finite in fp32, and so must scale * log2(e)")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype):
        raise ValueError("out must have q's shape and type")
    if out is not None and out.numel() and _meets_itself(out):
        raise ValueError("out must have batch entries and rows apart")
    if out is not None and any(_shares_memory(out, t) for t in (q, k, v)):
        raise ValueError("out must not share memory with q, k or v")
    if out is not None and any(t is not None and shares_memory(out, t) for t in (kv_lens, key_mask)):
        raise ValueError("out must not share memory with kv_lens or key_mask")
    if not use_kernels(q, k, v, kv_lens, key_mask, out):
        o, lse = cross_attention_reference(q, k, v, heads, heads_kv, kv_lens, key_mask, scale, True)
        o = o if out is None else out.copy_(o)
        return (o, lse) if return_lse else o
    # what the kernel does not take as it is: no rows, no keys, other strides, the first call on a device
    if Sk == 0 or q.numel() == 0:
        o = torch.zeros_like(q, memory_format=torch.contiguous_format) if out is None else out.zero_()
        lse = torch.full((B, heads, Sq), -math.inf, device=q.device, dtype=torch.float32) if return_lse else None
        return (o, lse) if return_lse else o
    status_word(q.device)
    if kv_lens is not None:
        kv_lens = kv_lens.clamp(0, Sk).to(torch.int32).contiguous()
    if out is not None and key_mask is not None and _shares_memory(out, key_mask):
        key_mask = key_mask.clone()  # beside out's rows
    got = launch("cross_attention", _strided(q), _strided(k), _strided(v), heads, heads_kv, kv_lens, key_mask, scale, out,
                 return_lse)
    if got is None:
        raise ValueError("cross_attention needs its tensors on one CUDA device and out with separate rows on 16 bytes")
    return got
