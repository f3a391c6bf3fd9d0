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
from .synth import Q8K_BYTES

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
        self._ref = ctypes.byref(self._c)

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
        self._ref = ctypes.byref(self._c)

    def rows(self, n_tokens: int):
        """The descriptor for a call of n_tokens rows."""
        self._c.n_tokens = n_tokens
        return self._ref


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
        self._ref = ctypes.byref(self._c)


class GpuAttn:
    """The attention-side operators of a handle."""

    def __init__(self, moe: GpuMoE):
        self.moe = moe
        self.index = moe.device
        self.device = torch.device("cuda", moe.device)
        self._lib = lib = _native.load_gpu()
        # a small call is as long as its way through Python: looked up once
        self._norm, self._read_q8, self._append = lib.lfm_gpu_add_rmsnorm, lib.lfm_gpu_q8k_read, lib.lfm_gpu_kv_append
        self._read, self._attend = lib.lfm_gpu_kv_read, lib.lfm_gpu_attn_forward

    def _stream(self) -> int:
        # the address alone: building torch's Stream object takes as long as a launch
        return torch._C._cuda_getCurrentRawStream(self.index)

    def _fail(self, st: int):
        raise MoEError(st, self._lib.lfm_gpu_moe_last_error(self.moe._h).decode(errors="replace"))

    def _rows(self, t: torch.Tensor, what: str, heads: Optional[int], dim: int, dtype) -> int:
        """Address of rows [tokens, heads, dim]."""
        shape = t.shape
        if len(shape) != 3 or not (t.is_contiguous() or (t.stride(2) == 1 and (shape[1] == 1 or t.stride(1) == dim))):
            raise ValueError(f"{what}: [tokens, heads, {dim}] with the heads of a token one behind the other")
        if shape[2] != dim or (heads is not None and shape[1] != heads) or t.get_device() != self.index or t.dtype != dtype:
            raise ValueError(f"{what} must be {dtype} [tokens, {heads or 'heads'}, {dim}] on {self.device}")
        return t.data_ptr()

    def _same_device(self, cache: KVPages, batch: KVBatch):
        if cache.index != self.index or batch.index != self.index:
            raise ValueError(f"cache and batch must be on {self.device}")

    # -- residual addition, RMSNorm, Q8_K ---------------------------------
    def add_rmsnorm(self, x: torch.Tensor, delta: Optional[torch.Tensor], weight: Optional[torch.Tensor], eps: float = 1e-5,
                    x_out: Optional[torch.Tensor] = None, xb_dtype: Optional[torch.dtype] = None, q8: bool = True
                    ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
        """(x + delta, its RMSNorm as xb_dtype or None, its RMSNorm as block_q8_K bytes [T, D / 256, 292] or None).
        x fp32 [T, D]; x_out may be x (in place)."""
        dev = self.index
        xp = _dense(x, "x", torch.float32, dev, 2)
        shape = T, D = x.shape
        dp = wp = bp = qp = xb = qb = None
        dt = bt = 0
        if delta is not None:
            dt = _type(delta.dtype, "delta")
            dp = _dense(delta, "delta", delta.dtype, dev, 2)
            if delta.shape != shape:
                raise ValueError("delta must have the shape of x")
        if weight is not None:
            wp = _dense(weight, "weight", torch.float32, dev, 1)
            if weight.shape[0] != D:
                raise ValueError(f"weight must have {D} values")
        if x_out is None:
            x_out = torch.empty_like(x)
            op = x_out.data_ptr()
        else:
            op = _dense(x_out, "x_out", torch.float32, dev, 2)
            if x_out.shape != shape:
                raise ValueError("x_out must have the shape of x")
        if xb_dtype is not None:
            bt = _type(xb_dtype, "xb_dtype")
            xb = x.new_empty(shape, dtype=xb_dtype)
            bp = xb.data_ptr()
        if q8:
            qb = x.new_empty((T, D // 256, Q8K_BYTES), dtype=torch.uint8)
            qp = qb.data_ptr()
        st = self._norm(self.moe._h, xp, dp, dt, T, D, wp, eps, op, bp, bt, qp, self._stream())
        if st:
            self._fail(st)
        return x_out, xb, qb

    def read_q8(self, q8: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """The values of block_q8_K rows [T, D / 256, 292] as [T, D]."""
        p = _dense(q8, "q8", torch.uint8, self.index, 3)
        T, n, size = q8.shape
        if size != Q8K_BYTES:
            raise ValueError(f"q8 must be [T, D / 256, {Q8K_BYTES}]")
        out = q8.new_empty((T, n * 256), dtype=dtype)
        st = self._read_q8(self.moe._h, p, T, n * 256, _type(dtype, "dtype"), out.data_ptr(), self._stream())
        if st:
            self._fail(st)
        return out

    # -- the cache ----------------------------------------------------------
    def append(self, cache: KVPages, batch: KVBatch, q: Optional[torch.Tensor], k: Optional[torch.Tensor],
               v: Optional[torch.Tensor], rope: Optional[Rope] = None, q_out: Optional[torch.Tensor] = None
               ) -> Optional[torch.Tensor]:
        """k and v [tokens, kv heads, dim] into the cache; returns q [tokens, heads, dim] normalised and rotated
        (into q_out, which may be q).  Either of q and (k, v) may be None."""
        self._same_device(cache, batch)
        first = q if q is not None else k
        if first is None or (k is None) != (v is None):
            raise ValueError("q, or k and v, or all three")
        T, dt, d = first.shape[0], first.dtype, cache.head_dim
        heads = qp = qs = op = os_ = kp = ks = vp = vs = 0
        if q is not None:
            qp, heads = self._rows(q, "q", None, d, dt), q.shape[1]
            qs = q.stride(0) if T != 1 else heads * d  # the stride of one row says nothing
            if q_out is None:
                q_out = q.new_empty(q.shape)
                op, os_ = q_out.data_ptr(), heads * d
            else:
                if q_out.shape[0] < T:
                    raise ValueError("q_out must have the rows of q")
                op = self._rows(q_out, "q_out", heads, d, dt)
                os_ = q_out.stride(0) if q_out.shape[0] != 1 else heads * d
        if k is not None:
            kp, vp = self._rows(k, "k", cache.n_kv_heads, d, dt), self._rows(v, "v", cache.n_kv_heads, d, dt)
            ks, vs = (k.stride(0), v.stride(0)) if T != 1 else (cache.n_kv_heads * d,) * 2
            if k.shape[0] != T or v.shape[0] != T:
                raise ValueError("q, k and v must have the same number of tokens")
        if rope is not None and (rope.norm_dim - {d} or (rope.index >= 0 and rope.index != self.index)):
            raise ValueError(f"q_norm and k_norm must have {d} values, rotation and norms be on {self.device}")
        st = self._append(self.moe._h, cache._ref, batch.rows(T), None if rope is None else rope._ref, _type(dt, "q"), heads, qp,
                          qs, op, os_, kp, ks, vp, vs, self._stream())
        if st:
            self._fail(st)
        return q_out

    def read(self, cache: KVPages, batch: KVBatch, n_tokens: int, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that the cache holds for the batch's n_tokens rows, [n_tokens, kv heads, dim] each."""
        self._same_device(cache, batch)
        kv = cache.pages.new_empty((2, n_tokens, cache.n_kv_heads, cache.head_dim), dtype=dtype)
        k, v = kv.unbind(0)
        st = self._read(self.moe._h, cache._ref, batch.rows(n_tokens), _type(dtype, "dtype"), k.data_ptr(), v.data_ptr(),
                        self._stream())
        if st:
            self._fail(st)
        return k, v

    # -- attention ------------------------------------------------------------
    def attend(self, cache: KVPages, batch: KVBatch, q: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
               window: int = 0, softcap: float = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q k) v over the cache, [tokens, heads, dim] like q (scale None: dim ** -0.5)."""
        self._same_device(cache, batch)
        d, dt = cache.head_dim, q.dtype
        qp = self._rows(q, "q", None, d, dt)
        T, heads, _ = shape = q.shape
        if out is None:
            out = q.new_empty(shape)
            op, os_ = out.data_ptr(), heads * d
        else:
            if out.shape[0] < T:
                raise ValueError("out must have the rows of q")
            op = self._rows(out, "out", heads, d, dt)
            os_ = out.stride(0) if out.shape[0] != 1 else heads * d
        st = self._attend(self.moe._h, cache._ref, batch.rows(T), heads, d ** -0.5 if scale is None else scale, causal, window,
                          softcap, _type(dt, "q"), qp, q.stride(0) if T != 1 else heads * d, op, os_, self._stream())
        if st:
            self._fail(st)
        return out

    def reserve(self):
        """Allocate attend's scratch now (needed before a stream capture)."""
        st = self._lib.lfm_gpu_attn_reserve(self.moe._h)
        if st:
            self._fail(st)
