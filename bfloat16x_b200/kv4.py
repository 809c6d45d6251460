"""Keys and values of attention held in 4 bits.

``Kv4Cache`` is the 4-bit counterpart of the decoder's bf16 cache tensors
(llama_e2e): ``append`` is the step between the qkv projection and attention
(rotary embedding of q and k, k and v quantised into the cache), ``attend`` the
attention over what the cache holds, for single tokens, a few tokens or whole
prompts, and ``read`` gives the held values back.  The reference has no cache of
its own.

Every 32 neighbouring channels of a position share a scale d and a minimum m
(bf16) and a value is d * code + m, code in 0..15: 5 bits per value, so a
position of one head takes 160 bytes at 128 channels where bf16 takes 512.
The blocks' byte order is described in csrc/bf16x_kv4.cuh.

Positions are device tensors, so that a captured step can move on: sequence b's
tokens are at ``pos0[b]``, ``pos0[b] + 1``, ...  A negative position is padding
(prompts of different lengths are padded on the left): it is not written, and
its rows come back as zeros.  A position at or past ``max_seq`` is skipped too
and reported by ``_lib.check_device_status``.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib

BLOCK = 16              # positions per block
GROUP = 32              # channels per scale


def kv4_blocks(batch: int, max_seq: int, kv_heads: int, head_dim: int, device=None) -> torch.Tensor:
    """Zeroed blocks [batch, kv_heads, ceil(max_seq / 16), 20 * head_dim] of a cache of ``max_seq`` positions."""
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    if batch < 1 or kv_heads < 1 or max_seq < 1:
        raise ValueError("batch, kv_heads and max_seq must be at least 1")
    return torch.zeros((batch, kv_heads, (max_seq + BLOCK - 1) // BLOCK, 20 * head_dim), dtype=torch.uint8,
                       device=device)


@lru_cache(maxsize=4096)
def _workspace_bytes(batch: int, tokens: int, heads: int, kv_heads: int, head_dim: int, max_seq: int) -> int:
    return int(_lib.lib().bf16x_kv4_attend_workspace_bytes(batch, tokens, heads, kv_heads, head_dim, max_seq))


class Kv4Cache:
    """The 4-bit cache of one layer over its ``blocks`` (``kv4_blocks``, or a slice of a larger tensor)."""

    __slots__ = ("blocks", "batch", "kv_heads", "max_seq", "head_dim", "device", "_index")

    def __init__(self, blocks: torch.Tensor, max_seq: int | None = None):
        if blocks.dtype is not torch.uint8 or blocks.dim() != 4 or not blocks.is_contiguous():
            raise ValueError("blocks must be a contiguous uint8 tensor [batch, kv_heads, blocks, 20 * head_dim]")
        self.blocks = blocks
        self.batch, self.kv_heads, n, size = blocks.shape
        if size != 1280 and size != 2560:
            raise ValueError(f"head_dim must be 64 or 128 (blocks of 1280 or 2560 bytes), got blocks of {size} bytes")
        self.head_dim = size // 20
        self.max_seq = n * BLOCK if max_seq is None else int(max_seq)
        if not (n - 1) * BLOCK < self.max_seq <= n * BLOCK:
            raise ValueError(f"{n} blocks hold {(n - 1) * BLOCK + 1}..{n * BLOCK} positions, not {self.max_seq}")
        self.device = blocks.device
        self._index = self.device.index

    @classmethod
    def empty(cls, batch: int, max_seq: int, kv_heads: int, head_dim: int, device=None) -> "Kv4Cache":
        return cls(kv4_blocks(batch, max_seq, kv_heads, head_dim, device), max_seq)

    def nbytes(self) -> int:
        return self.blocks.numel()

    def _pos(self, pos0: torch.Tensor) -> int:
        """The stride of the positions of the sequences (0: one for all)."""
        if pos0.dtype is not torch.int64 or pos0.device != self.device:
            raise ValueError("pos0 must be an int64 tensor on the cache's device")
        if pos0.numel() == 1:
            return 0
        if pos0.dim() != 1 or pos0.shape[0] != self.batch:
            raise ValueError(f"pos0 must hold one position, or one for each of {self.batch} sequences")
        return pos0.stride(0)

    def _check(self, x: torch.Tensor, name: str) -> None:
        if x.dtype is not torch.bfloat16:
            raise ValueError(f"{name} must be bf16")
        if x.device != self.device or self._index is None:
            _lib.require_cuda(x, name)
            raise ValueError(f"{name} must be on the cache's device")

    def append(self, qkv: torch.Tensor, pos0: torch.Tensor, heads: int, cos: torch.Tensor | None = None,
               sin: torch.Tensor | None = None) -> torch.Tensor:
        """qkv [batch, T, (heads + 2 kv_heads) * head_dim] (bf16): q and k
        turned pairwise by the angles of their positions (``cos``/``sin``
        fp32 [>= max_seq, head_dim / 2]; None: not turned), k and v written
        into the cache at pos0[b] + t.  Returns q [batch, T, heads, head_dim]
        (zeros where the position lies outside the cache)."""
        self._check(qkv, "qkv")
        B, KV, D = self.batch, self.kv_heads, self.head_dim
        if heads < 0 or qkv.dim() != 3 or qkv.shape[0] != B or qkv.shape[2] != (heads + 2 * KV) * D:
            raise ValueError(f"qkv must be [{B}, T, (heads + {2 * KV}) * {D}], got {tuple(qkv.shape)} for {heads} heads")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin go together")
        c = s = None
        if cos is not None:
            for a in (cos, sin):
                if (a.dtype is not torch.float32 or a.dim() != 2 or a.shape[1] != D // 2 or a.shape[0] < self.max_seq
                        or not a.is_contiguous() or a.device != self.device):
                    raise ValueError(f"cos and sin must be contiguous fp32 [>= {self.max_seq}, {D // 2}] on the cache's device")
            c, s = cos.data_ptr(), sin.data_ptr()
        stride = self._pos(pos0)
        ld_b, ld_t, one = qkv.stride()
        if one != 1 or (ld_b | ld_t) % 8 or qkv.data_ptr() % 16:
            qkv = qkv.clone(memory_format=torch.contiguous_format)
            ld_b, ld_t, _ = qkv.stride()
        T = qkv.shape[1]
        q = torch.empty((B, T, heads, D), dtype=torch.bfloat16, device=self.device)
        _lib.call_on(self._index, "bf16x_kv4_append", qkv.data_ptr(), ld_b, ld_t, B, T, heads, KV, D, pos0.data_ptr(),
                     stride, c, s, q.data_ptr(), self.blocks.data_ptr(), self.max_seq)
        return q

    def read(self, pos0: torch.Tensor, count: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [batch, count, kv_heads, head_dim] bf16: what the cache
        holds at positions pos0[b] .. pos0[b] + count - 1 (zeros outside it)."""
        _lib.require_cuda(self.blocks, "blocks")
        if count < 0:
            raise ValueError("count must not be negative")
        stride = self._pos(pos0)
        shape = (self.batch, count, self.kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        _lib.call_on(self._index, "bf16x_kv4_read", self.blocks.data_ptr(), self.max_seq, self.batch, count,
                     self.kv_heads, self.head_dim, pos0.data_ptr(), stride, k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, q: torch.Tensor, pos0: torch.Tensor, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of q [batch, T, heads, head_dim] (bf16, heads a
        multiple of kv_heads) over the cache: the row at position pos0[b] + t
        sees positions 0 .. pos0[b] + t.  scale: default head_dim ** -0.5.
        Returns bf16 like q (zeros for a row that sees nothing or whose
        position lies past the cache).  The cache has no gradient."""
        self._check(q, "q")
        KV, D = self.kv_heads, self.head_dim
        shape = q.shape
        if len(shape) != 4 or shape[0] != self.batch or shape[3] != D or shape[2] % KV or shape[2] == 0:
            raise ValueError(f"q must be [{self.batch}, T, a multiple of {KV}, {D}], got {tuple(shape)}")
        stride = self._pos(pos0)
        B, T, H, _ = shape
        s0, s1, s2, one = q.stride()
        if one != 1 or (s0 | s1 | s2) % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            s0, s1, s2, _ = q.stride()
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)        # (half the time of torch.empty)
        elif (out.shape != shape or out.dtype is not torch.bfloat16 or not out.is_contiguous()
              or out.device != self.device or out.data_ptr() % 16):
            raise ValueError("out must be a contiguous, 16-byte aligned bf16 tensor of q's shape")
        elif out.numel():               # rows are written while others are still read
            at, last = q.data_ptr(), (B - 1) * s0 + (T - 1) * s1 + (H - 1) * s2 + D
            if at < out.data_ptr() + 2 * out.numel() and out.data_ptr() < at + 2 * last:
                raise ValueError("out must not overlap q")
        # a workspace of its own for every call (and every captured graph): calls may overlap on several streams
        need = _workspace_bytes(B, T, H, KV, D, self.max_seq)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        _lib.call_on(self._index, "bf16x_kv4_attend", q.data_ptr(), s0, s1, s2, B, T, H, KV, D, pos0.data_ptr(), stride,
                     D ** -0.5 if scale is None else float(scale), self.blocks.data_ptr(), self.max_seq, out.data_ptr(),
                     None if ws is None else ws.data_ptr(), need)
        return out


__all__ = ["Kv4Cache", "kv4_blocks", "BLOCK", "GROUP"]
