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


class Kv4Cache:
    """The 4-bit cache of one layer over its ``blocks`` (``kv4_blocks``, or a slice of a larger tensor)."""

    __slots__ = ("blocks", "batch", "kv_heads", "max_seq", "head_dim")

    def __init__(self, blocks: torch.Tensor, max_seq: int | None = None):
        if blocks.dtype != torch.uint8 or blocks.dim() != 4 or not blocks.is_contiguous():
            raise ValueError("blocks must be a contiguous uint8 tensor [batch, kv_heads, blocks, 20 * head_dim]")
        self.blocks = blocks
        self.batch, self.kv_heads, n, size = blocks.shape
        if size != 1280 and size != 2560:
            raise ValueError(f"head_dim must be 64 or 128 (blocks of 1280 or 2560 bytes), got blocks of {size} bytes")
        self.head_dim = size // 20
        self.max_seq = n * BLOCK if max_seq is None else int(max_seq)
        if not (n - 1) * BLOCK < self.max_seq <= n * BLOCK:
            raise ValueError(f"{n} blocks hold {(n - 1) * BLOCK + 1}..{n * BLOCK} positions, not {self.max_seq}")

    @classmethod
    def empty(cls, batch: int, max_seq: int, kv_heads: int, head_dim: int, device=None) -> "Kv4Cache":
        return cls(kv4_blocks(batch, max_seq, kv_heads, head_dim, device), max_seq)

    def nbytes(self) -> int:
        return self.blocks.numel()

    def _pos(self, pos0: torch.Tensor) -> int:
        """The stride of the positions of the sequences (0: one for all)."""
        if pos0.dtype != torch.int64 or pos0.device != self.blocks.device:
            raise ValueError("pos0 must be an int64 tensor on the cache's device")
        n = pos0.numel()
        if n == 1:
            return 0
        if pos0.dim() != 1 or n != self.batch:
            raise ValueError(f"pos0 must hold one position, or one for each of {self.batch} sequences")
        return pos0.stride(0)

    def _check(self, x: torch.Tensor, name: str) -> None:
        _lib.require_cuda(x, name)
        if x.device != self.blocks.device:
            raise ValueError(f"{name} must be on the cache's device")
        if x.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bf16")

    def _call(self, name: str, *args) -> None:
        """The entry point on the cache's device and its current stream."""
        dev = self.blocks.device
        if torch.cuda.current_device() == dev.index:
            _lib.check(getattr(_lib.lib(), name)(*args, torch.cuda.current_stream().cuda_stream), name)
        else:
            with torch.cuda.device(dev):
                _lib.check(getattr(_lib.lib(), name)(*args, torch.cuda.current_stream().cuda_stream), name)

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
        if cos is not None:
            for a in (cos, sin):
                if (a.dtype != torch.float32 or a.dim() != 2 or a.shape[1] != D // 2 or a.shape[0] < self.max_seq
                        or not a.is_contiguous() or a.device != qkv.device):
                    raise ValueError(f"cos and sin must be contiguous fp32 [>= {self.max_seq}, {D // 2}] on the cache's device")
        stride = self._pos(pos0)
        if qkv.stride(2) != 1 or qkv.stride(0) % 8 or qkv.stride(1) % 8 or qkv.data_ptr() % 16:
            qkv = qkv.clone(memory_format=torch.contiguous_format)
        T = qkv.shape[1]
        q = torch.empty((B, T, heads, D), dtype=torch.bfloat16, device=qkv.device)
        self._call("bf16x_kv4_append", qkv.data_ptr(), qkv.stride(0), qkv.stride(1), B, T, heads, KV, D,
                   pos0.data_ptr(), stride, _lib.ptr(cos), _lib.ptr(sin), q.data_ptr(), self.blocks.data_ptr(),
                   self.max_seq)
        return q

    def read(self, pos0: torch.Tensor, count: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [batch, count, kv_heads, head_dim] bf16: what the cache
        holds at positions pos0[b] .. pos0[b] + count - 1 (zeros outside it)."""
        _lib.require_cuda(self.blocks, "blocks")
        if count < 0:
            raise ValueError("count must not be negative")
        stride = self._pos(pos0)
        shape = (self.batch, count, self.kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.blocks.device)
        v = torch.empty_like(k)
        self._call("bf16x_kv4_read", self.blocks.data_ptr(), self.max_seq, self.batch, count, self.kv_heads,
                   self.head_dim, pos0.data_ptr(), stride, k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, q: torch.Tensor, pos0: torch.Tensor, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of q [batch, T, heads, head_dim] (bf16, heads a
        multiple of kv_heads) over the cache: the row at position pos0[b] + t
        sees positions 0 .. pos0[b] + t.  scale: default head_dim ** -0.5.
        Returns bf16 like q (zeros for a row that sees nothing)."""
        self._check(q, "q")
        B, KV, D = self.batch, self.kv_heads, self.head_dim
        if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D or q.shape[2] % KV or q.shape[2] == 0:
            raise ValueError(f"q must be [{B}, T, a multiple of {KV}, {D}], got {tuple(q.shape)}")
        stride = self._pos(pos0)
        s = q.stride()
        if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            s = q.stride()
        T, H = q.shape[1], q.shape[2]
        if out is None:
            out = torch.empty((B, T, H, D), dtype=torch.bfloat16, device=q.device)
        elif (out.shape != q.shape or out.dtype != torch.bfloat16 or not out.is_contiguous() or out.device != q.device
              or out.data_ptr() % 16):
            raise ValueError("out must be a contiguous, 16-byte aligned bf16 tensor of q's shape")
        # a workspace of its own for every call (and every captured graph): calls may overlap on several streams
        need = _lib.lib().bf16x_kv4_attend_workspace_bytes(B, T, H, KV, D, self.max_seq)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        self._call("bf16x_kv4_attend", q.data_ptr(), s[0], s[1], s[2], B, T, H, KV, D, pos0.data_ptr(), stride,
                   D ** -0.5 if scale is None else float(scale), self.blocks.data_ptr(), self.max_seq, out.data_ptr(),
                   _lib.ptr(ws), need)
        return out


__all__ = ["Kv4Cache", "kv4_blocks", "BLOCK", "GROUP"]
