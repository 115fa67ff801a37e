"""ctypes face of the paged 8-bit cache of keys and values (sfq_kv_cache_append, sfq_kv_cache_attention)."""
from __future__ import annotations

import ctypes as C
import struct
from dataclasses import dataclass

import torch

from . import KvCacheDesc, RotaryDesc, check, lib, ptr
from .linear import SAME_DEVICE, on_device, raw_stream

HEAD_DIM = 128
_INT = torch.int32
_POOL = ("k", "v", "k_scale", "v_scale")
_FIELDS = struct.Struct("4P4i3P4i")  # sfq_kv_cache; packed at once, which takes a quarter of the time of ctypes' constructor


@dataclass
class Sequences:
    """The sequences of a step. page_table int32 [batch, max_pages], seq_len int32 [batch] (new tokens included), row_start int32
    [batch + 1]; max_new and max_len: the most new tokens of a sequence and the longest sequence, estimates that size the launch."""
    page_table: torch.Tensor
    seq_len: torch.Tensor
    row_start: torch.Tensor
    max_new: int
    max_len: int


@dataclass(frozen=True)
class Rotary:
    """What happens to q and k on the way into the cache: head norm (bf16 [128] weights) and rotation (fp32 [table_rows, rotary_dim / 2]
    tables) at `position` int32 [rows], or at each token's place in its sequence."""
    cos: torch.Tensor | None = None
    sin: torch.Tensor | None = None
    position: torch.Tensor | None = None
    q_norm: torch.Tensor | None = None
    k_norm: torch.Tensor | None = None
    eps: float = 1e-6

    def __post_init__(self):
        for name, dtype in (("cos", torch.float32), ("sin", torch.float32), ("position", torch.int32), ("q_norm", torch.bfloat16), ("k_norm", torch.bfloat16)):
            t = getattr(self, name)
            if t is not None and t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype}")
        if (self.cos is None) != (self.sin is None) or (self.cos is not None and (self.cos.dim() != 2 or self.cos.shape != self.sin.shape)):
            raise ValueError("cos and sin come together, [table_rows, rotary_dim / 2] each")
        for t in (self.q_norm, self.k_norm):
            if t is not None and t.shape != (HEAD_DIM,):
                raise ValueError("norm weights have 128 elements")
        devices = {t.get_device() for t in (self.cos, self.sin, self.position, self.q_norm, self.k_norm) if t is not None}
        if len(devices) > 1:
            raise ValueError("the tables, positions and norm weights lie on one device")
        shape = self.cos.shape if self.cos is not None else (0, 0)
        rows, half = shape
        object.__setattr__(self, "device", devices.pop() if devices else None)
        object.__setattr__(self, "desc", RotaryDesc(ptr(self.cos), ptr(self.sin), ptr(self.position), rows, 2 * half, ptr(self.q_norm), ptr(self.k_norm), self.eps))
        object.__setattr__(self, "_shape", shape)
        object.__setattr__(self, "_held", [(t, t.data_ptr()) for t in (self.cos, self.sin, self.position, self.q_norm, self.k_norm) if t is not None])

    def _desc_now(self) -> RotaryDesc:
        for t, at in self._held:
            if t.data_ptr() != at:  # the tensor has got other memory
                self.__post_init__()
                break
        else:
            if self.cos is not None and self.cos.shape != self._shape:
                self.__post_init__()
        return self.desc


class KvCache:
    """Pages of keys and values in e4m3 with one scale per (page, head): k uint8 [pages, kv_heads, page_size, 128], v uint8 [pages,
    kv_heads, 128, page_size], scales fp32 [pages, kv_heads]. The tensors are the caller's; `KvCache.empty` makes them. They may be
    replaced, all four for a pool of another size: a call takes them as they then are."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._check_pool()

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        if name in _POOL:
            object.__setattr__(self, "_pool", None)

    def _check_pool(self) -> None:
        k, v, k_scale, v_scale = self.k, self.v, self.k_scale, self.v_scale
        pages, kv_heads, page_size, dim = k.shape
        if k.dtype != torch.uint8 or v.dtype != torch.uint8 or v.shape != (pages, kv_heads, dim, page_size):
            raise ValueError("k must be uint8 [pages, kv_heads, page_size, 128] and v [pages, kv_heads, 128, page_size]")
        for t in (k_scale, v_scale):
            if t.dtype != torch.float32 or t.shape != (pages, kv_heads):
                raise ValueError("scales must be fp32 [pages, kv_heads]")
        if len({t.device for t in (k, v, k_scale, v_scale)}) != 1:
            raise ValueError("the pools and their scales lie on one device")
        places = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (k, v, k_scale, v_scale))
        if any(end > start for (_, end), (start, _) in zip(places, places[1:])):
            raise ValueError("k, v and their scales lie apart")
        self.kv_heads, self.device, self._device = kv_heads, k.device, k.get_device()
        self._pool, self._shape = (ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), pages, page_size, kv_heads, dim), k.shape

    @staticmethod
    def empty(pages: int, kv_heads: int, page_size: int = 64, device="cuda") -> "KvCache":
        k = torch.zeros((pages, kv_heads, page_size, HEAD_DIM), dtype=torch.uint8, device=device)
        v = torch.zeros((pages, kv_heads, HEAD_DIM, page_size), dtype=torch.uint8, device=device)
        return KvCache(k, v, *(torch.zeros((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)))

    def _pool_now(self) -> tuple:
        pool, k = self._pool, self.k
        if pool is None or k.data_ptr() != pool[0] or self.v.data_ptr() != pool[1] or self.k_scale.data_ptr() != pool[2] or self.v_scale.data_ptr() != pool[3] or k.shape != self._shape:
            self._check_pool()  # a tensor was replaced, or has got other memory
            pool = self._pool
        return pool

    def _desc(self, s: Sequences, pool: tuple | None = None) -> KvCacheDesc:
        if pool is None:
            pool = self._pool_now()
        t, n, r = s.page_table, s.seq_len, s.row_start
        if t.dtype != _INT or n.dtype != _INT or r.dtype != _INT:
            raise ValueError("page_table, seq_len and row_start must be int32")
        batch, max_pages = t.shape
        if n.shape != (batch,) or r.shape != (batch + 1,) or not (t.is_contiguous() and n.is_contiguous() and r.is_contiguous()):
            raise ValueError("seq_len has an entry per sequence, row_start one more; all are contiguous")
        if not t.get_device() == n.get_device() == r.get_device() == self._device:
            raise ValueError("the sequences' tensors lie on the cache's device")
        return KvCacheDesc.from_buffer_copy(_FIELDS.pack(*pool, t.data_ptr(), n.data_ptr(), r.data_ptr(), batch, max_pages, s.max_new, s.max_len))

    def _pitch(self, name: str, t: torch.Tensor, rows: int | None, cols: int) -> int:
        return self._rows_and_pitch(name, t, rows, cols)[1]

    def _rows_and_pitch(self, name: str, t: torch.Tensor, rows: int | None, cols: int) -> tuple[int, int]:
        shape, stride = t.shape, t.stride()
        if t.dtype != torch.bfloat16 or len(shape) != 2 or shape[1] != cols or stride[1] != 1 or t.get_device() != self._device or rows not in (None, shape[0]):
            raise ValueError(f"{name} must be bf16 [{'rows' if rows is None else rows}, {cols}] with contiguous rows, on the cache's device")
        if shape[0] <= 1:
            return shape[0], cols  # a single row may have any stride
        if stride[0] < cols:
            raise ValueError(f"{name}'s rows overlap: they lie {stride[0]} elements apart and have {cols}")
        if stride[0] >= 1 << 31:
            raise ValueError(f"{name}'s rows lie {stride[0]} elements apart; the library takes a pitch of 32 bits")
        return shape[0], stride[0]

    def append(self, s: Sequences, qkv: torch.Tensor, heads: int, q_out: torch.Tensor | None = None, rotary: Rotary | None = None) -> torch.Tensor:
        """Stores k and v of the fused projection qkv [rows, (heads + 2 kv_heads) * 128] and returns q, normed and rotated
        (q_out [rows, heads * 128]; pass a view of qkv's first columns to have it in place)."""
        pool = self._pool_now()
        rows, ld = self._rows_and_pitch("qkv", qkv, None, (heads + 2 * self.kv_heads) * HEAD_DIM)
        ld_out = heads * HEAD_DIM
        if q_out is None:
            q_out = qkv.new_empty((rows, ld_out))
        else:
            ld_out = self._pitch("q_out", q_out, rows, ld_out)
        rotation = None
        if rotary is not None:
            rotation = rotary._desc_now()
            if rotary.position is not None and rotary.position.shape != (rows,):
                raise ValueError("position has an entry per row")
            if rotary.device not in (None, self._device):
                raise ValueError("the rotation's tensors lie on the cache's device")
        q = qkv.data_ptr()
        k = q + heads * HEAD_DIM * 2
        here = on_device(self._device)
        args = (C.byref(self._desc(s, pool)), C.byref(rotation) if rotation is not None else None, q, ld, q_out.data_ptr(), ld_out,
                heads, k, k + self.kv_heads * HEAD_DIM * 2, ld, rows, raw_stream(self._device))
        if here is SAME_DEVICE:
            status = lib.sfq_kv_cache_append(*args)
        else:
            with here:
                status = lib.sfq_kv_cache_append(*args)
        if status:
            check(status)
        return q_out

    def attention(self, s: Sequences, q: torch.Tensor, heads: int, out: torch.Tensor | None = None, scale: float = 0.0) -> torch.Tensor:
        """softmax(q K^T scale) V of the new tokens' q [rows, heads * 128] over the cache, causal among them; scale 0 means 1 / sqrt(128).
        The workspace is the call's own, so that calls on several streams and captured graphs share none."""
        pool = self._pool_now()
        rows, ld = self._rows_and_pitch("q", q, None, heads * HEAD_DIM)
        ld_out = heads * HEAD_DIM
        if out is None:
            out = q.new_empty((rows, ld_out))
        else:
            ld_out = self._pitch("out", out, rows, ld_out)
        with on_device(self._device):
            desc, n = self._desc(s, pool), C.c_size_t()
            check(lib.sfq_kv_cache_attention_workspace_bytes(C.byref(desc), heads, rows, C.byref(n)))
            ws = torch.empty(n.value, dtype=torch.uint8, device=self.device) if n.value else None
            status = lib.sfq_kv_cache_attention(C.byref(desc), q.data_ptr(), ld, out.data_ptr(), ld_out, heads, rows, scale, ws.data_ptr() if n.value else None,
                                                n.value, raw_stream(self._device))
        if status:
            check(status)
        return out
