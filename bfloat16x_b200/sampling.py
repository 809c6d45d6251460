"""Drawing the next token from logits: temperature, top-k, top-p and min-p with
given random numbers (the decoder's step after lm_head; the reference has no
decoder of its own)."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from ._lib import BF16X_DTYPE_BF16, BF16X_DTYPE_F32

_DT = {torch.bfloat16: BF16X_DTYPE_BF16, torch.float32: BF16X_DTYPE_F32}


@dataclass
class SamplingParams:
    """The settings of ``sample``, each a number or a tensor of one value per row."""
    temperature: float | torch.Tensor = 1.0
    top_k: int | torch.Tensor = 0
    top_p: float | torch.Tensor = 1.0
    min_p: float | torch.Tensor = 0.0


def _setting(x, name: str, dtype: torch.dtype, logits: torch.Tensor):
    """(device pointer or None, value) of a setting given as a number or as a tensor of one value per row."""
    if not isinstance(x, torch.Tensor):
        return None, x
    if x.dtype != dtype or x.dim() != 1 or x.shape[0] != logits.shape[0] or not x.is_contiguous() \
            or x.device != logits.device:
        raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor [{logits.shape[0]}] on the logits' device")
    return x.data_ptr(), 0


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Tokens [rows] (int64) drawn from logits [rows, vocab] (bf16 or fp32).

    u: fp32 [rows] in [0, 1), the random numbers.  Each setting is one number
    or a tensor with one value per row (fp32; top_k int32).  The tokens of a
    row are ordered by logit, ties by index, and weigh exp((logit - max) /
    temperature); then

    * ``top_k`` > 0 keeps the first k of the order,
    * ``top_p`` < 1 keeps the shortest prefix whose weight reaches top_p times
      that of what top_k kept (at least one token),
    * ``min_p`` > 0 keeps tokens of at least min_p times the largest weight,

    and the token drawn is the first kept one, in index order, whose running
    weight exceeds u times the kept weight.  temperature <= 0 or top_k == 1
    takes the largest logit (the lowest index among equal ones).  NaN logits
    count as -infinity, and a row with no logit above -infinity gives -1.
    Weights are summed exactly, so equal inputs always give equal tokens.
    """
    _lib.require_cuda(logits, "logits")
    if logits.dim() != 2 or logits.dtype not in _DT:
        raise ValueError("logits must be [rows, vocab] in bf16 or fp32")
    B, V = logits.shape
    if V == 0:
        raise ValueError("logits must have at least one token")
    if u.dtype != torch.float32 or u.dim() != 1 or u.shape[0] != B or not u.is_contiguous() or u.device != logits.device:
        raise ValueError(f"u must be a contiguous fp32 tensor [{B}] on the logits' device")
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=logits.device)
    elif out.dtype != torch.int64 or out.shape != (B,) or not out.is_contiguous() or out.device != logits.device:
        raise ValueError(f"out must be a contiguous int64 tensor [{B}] on the logits' device")
    t, t0 = _setting(temperature, "temperature", torch.float32, logits)
    k, k0 = _setting(top_k, "top_k", torch.int32, logits)
    p, p0 = _setting(top_p, "top_p", torch.float32, logits)
    m, m0 = _setting(min_p, "min_p", torch.float32, logits)
    if B and (logits.stride(1) != 1 or logits.stride(0) < V):
        logits = logits.clone(memory_format=torch.contiguous_format)
    _lib.call_on(logits.device.index, "bf16x_sample", logits.data_ptr(), _DT[logits.dtype], max(logits.stride(0), V), B, V,
                 u.data_ptr(), t, float(t0), k, max(0, min(int(k0), 0x7FFFFFFF)), p, float(p0), m, float(m0),
                 out.data_ptr())
    return out


__all__ = ["sample", "SamplingParams"]
