"""Python host API over include/lfm_gpu_attn.h on torch tensors of the handle's device.

What an lfm2moe layer does before its MoE FFN (``laii_b200.moe``): the residual's addition with RMSNorm and
Q8_K rows, q/k normalisation and rotation with keys and values into a paged 4-bit cache, and grouped-query
attention over it.  Calls run on torch's current stream, asynchronously; errors come back as ``MoEError`` with
the library's status code, wrong tensors as ``ValueError``; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _native
from .moe import GpuMoE, MoEError

GGML_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _type(dtype: torch.dtype, what: str) -> int:
    t = GGML_TYPE.get(dtype)
    if t is None:
        raise ValueError(f"{what}: {dtype} (float32, float16 or bfloat16)")
    return t


def _dense(t: Optional[torch.Tensor], what: str, dtype: torch.dtype, index: int, ndim: int) -> Optional[int]:
    """The address of a contiguous tensor on CUDA device `index` (None stays None)."""
    if t is None:
        return None
    if t.dtype != dtype or t.get_device() != index or t.dim() != ndim or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {ndim}-d {dtype} tensor on CUDA device {index}")
    return t.data_ptr()


class KVPages:
    """One layer's pool of 4-bit cache pages over a uint8 tensor that the caller owns (layout: lfm_gpu_kv_t)."""

    def __init__(self, pages: torch.Tensor, page_tokens: int, n_kv_heads: int, head_dim: int):
        size = self.page_bytes(page_tokens, n_kv_heads, head_dim)
        if size == 0:
            raise ValueError(f"no cache of {page_tokens}-token pages and {n_kv_heads} heads of {head_dim}")
        if pages.dtype != torch.uint8 or not pages.is_cuda or not pages.is_contiguous() or pages.numel() % size:
            raise ValueError(f"pages must be a contiguous uint8 CUDA tensor of whole {size}-byte pages")
        self.pages, self.page_tokens, self.n_kv_heads, self.head_dim = pages, page_tokens, n_kv_heads, head_dim
        self.n_pages = pages.numel() // size
        self.index = pages.get_device()
        self._c = _native.Kv(pages.data_ptr(), self.n_pages, page_tokens, n_kv_heads, head_dim)
        self._at = ctypes.addressof(self._c)

    @staticmethod
    def page_bytes(page_tokens: int, n_kv_heads: int, head_dim: int) -> int:
        """Bytes of a page, 0 for a shape that is not supported."""
        return _native.load_gpu().lfm_gpu_kv_page_bytes(page_tokens, n_kv_heads, head_dim)

    @classmethod
    def empty(cls, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, device="cuda") -> "KVPages":
        size = cls.page_bytes(page_tokens, n_kv_heads, head_dim)
        return cls(torch.empty(n_pages, size, dtype=torch.uint8, device=device), page_tokens, n_kv_heads, head_dim)


class KVBatch:
    """A ragged batch: int32 device tensors q_start [n + 1], kv_len [n] and page_table [n, pages], read when a call
    runs (lfm_gpu_kv_batch_t).  max_kv_len plans the work; any value is safe."""

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, max_kv_len: int = 0):
        n, dev = kv_len.numel(), kv_len.get_device()
        if not kv_len.is_cuda or q_start.numel() != n + 1 or page_table.dim() != 2 or page_table.shape[0] != n:
            raise ValueError("q_start [n + 1], kv_len [n] and page_table [n, pages] on one CUDA device")
        self.index = dev
        self._keep = (q_start, kv_len, page_table)
        self._c = _native.KvBatch(n, 0, page_table.shape[1], max_kv_len, _dense(q_start, "q_start", torch.int32, dev, 1),
                                  _dense(kv_len, "kv_len", torch.int32, dev, 1),
                                  _dense(page_table, "page_table", torch.int32, dev, 2))
        self._at = ctypes.addressof(self._c)

    def rows(self, n_tokens: int):
        """The descriptor for a call of n_tokens rows, for the C-ABI."""
        self._c.n_tokens = n_tokens
        return ctypes.byref(self._c)


class Rope:
    """Per-head norms and the rotation that append applies (lfm_gpu_rope_t): cos and sin fp32 [positions, rot_dim / 2]."""

    def __init__(self, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, pairs: bool = False,
                 q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-5):
        if (cos is None) != (sin is None) or (cos is not None and cos.shape != sin.shape):
            raise ValueError("cos and sin come together, of one shape")
        given = [t for t in (cos, q_norm, k_norm) if t is not None]
        dev = given[0].get_device() if given else -1
        self._keep = (cos, sin, q_norm, k_norm)
        self.norm_dim = {t.numel() for t in (q_norm, k_norm) if t is not None}
        self._c = _native.Rope(_dense(cos, "cos", torch.float32, dev, 2), _dense(sin, "sin", torch.float32, dev, 2),
                               0 if cos is None else cos.shape[0], 0 if cos is None else 2 * cos.shape[1], int(pairs), eps,
                               _dense(q_norm, "q_norm", torch.float32, dev, 1), _dense(k_norm, "k_norm", torch.float32, dev, 1))
        self.index = dev
        self._at = ctypes.addressof(self._c)


class GpuAttn:
    """The attention-side operators of a handle."""

    def __init__(self, moe: GpuMoE):
        self.moe = moe
        self.index = moe.device
        self.device = torch.device("cuda", moe.device)
        self._lib, self._py = _native.load_gpu(), _native.load_attn_py()

    def _stream(self) -> int:
        """torch's current stream, for calls of the C-ABI itself."""
        return torch._C._cuda_getCurrentRawStream(self.index)

    def _handle(self) -> int:
        h = self.moe._h
        if h is None:
            raise ValueError("the handle is closed")
        return h.value

    def _done(self, result):
        """What a call of lfm_attn_py returned: its outputs, or a status."""
        if type(result) is int:
            raise MoEError(result, self._lib.lfm_gpu_moe_last_error(self.moe._h).decode(errors="replace"))
        return result

    def _same_device(self, cache: KVPages, batch: KVBatch):
        if cache.index != self.index or batch.index != self.index:
            raise ValueError(f"cache and batch must be on {self.device}")

    # -- residual addition, RMSNorm, Q8_K ---------------------------------
    def add_rmsnorm(self, x: torch.Tensor, delta: Optional[torch.Tensor], weight: Optional[torch.Tensor], eps: float = 1e-5,
                    x_out: Optional[torch.Tensor] = None, xb_dtype: Optional[torch.dtype] = None, q8: bool = True
                    ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
        """(x + delta, its RMSNorm as xb_dtype or None, its RMSNorm as block_q8_K bytes [T, D / 256, 292] or None).
        x fp32 [T, D]; x_out may be x (in place)."""
        return self._done(self._py.add_rmsnorm(self._handle(), self.index, x, delta, weight, eps, x_out,
                                               -1 if xb_dtype is None else _type(xb_dtype, "xb_dtype"), q8))

    def read_q8(self, q8: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """The values of block_q8_K rows [T, D / 256, 292] as [T, D]."""
        return self._done(self._py.read_q8(self._handle(), self.index, q8, _type(dtype, "dtype")))

    # -- the cache ----------------------------------------------------------
    def append(self, cache: KVPages, batch: KVBatch, q: Optional[torch.Tensor], k: Optional[torch.Tensor],
               v: Optional[torch.Tensor], rope: Optional[Rope] = None, q_out: Optional[torch.Tensor] = None
               ) -> Optional[torch.Tensor]:
        """k and v [tokens, kv heads, dim] into the cache; returns q [tokens, heads, dim] normalised and rotated
        (into q_out, which may be q).  Either of q and (k, v) may be None."""
        self._same_device(cache, batch)
        if rope is not None and (rope.norm_dim - {cache.head_dim} or (rope.index >= 0 and rope.index != self.index)):
            raise ValueError(f"q_norm and k_norm must have {cache.head_dim} values, rotation and norms be on {self.device}")
        return self._done(self._py.append(self._handle(), self.index, cache._at, batch._at, None if rope is None else rope._at,
                                          q, k, v, q_out))

    def read(self, cache: KVPages, batch: KVBatch, n_tokens: int, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that the cache holds for the batch's n_tokens rows, [n_tokens, kv heads, dim] each."""
        self._same_device(cache, batch)
        return self._done(self._py.read(self._handle(), self.index, cache._at, batch._at, n_tokens, _type(dtype, "dtype")))

    # -- attention ------------------------------------------------------------
    def attend(self, cache: KVPages, batch: KVBatch, q: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
               window: int = 0, softcap: float = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q k) v over the cache, [tokens, heads, dim] like q (scale None: dim ** -0.5)."""
        self._same_device(cache, batch)
        return self._done(self._py.attend(self._handle(), self.index, cache._at, batch._at, q,
                                          cache.head_dim ** -0.5 if scale is None else scale, causal, window, softcap, out))

    def reserve(self):
        """Allocate attend's scratch now (needed before a stream capture)."""
        self._done(self._lib.lfm_gpu_attn_reserve(self._handle()) or None)
