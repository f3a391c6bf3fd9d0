"""The attention-side operators in 64 bits, from their definitions (include/lfm_gpu_attn.h), on CPU tensors."""
import math

import torch


def unpack_head(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """codes uint8 [..., D / 2], scales fp16 [..., D / 32] -> float64 values [..., D]."""
    d = 2 * codes.shape[-1]
    out = torch.empty(*codes.shape[:-1], d, dtype=torch.float64)
    for i in range(d):
        word, nib = (i % 32) // 4, (i % 64) // 32 * 4 + i % 4
        byte = (i // 64) * 32 + 4 * word + nib // 2
        c = (codes[..., byte] >> (4 * (nib % 2))) & 15
        out[..., i] = (c.double() - 8) * scales[..., i // 32].double()
    return out


def split_page(pages: torch.Tensor, P: int, hkv: int, D: int):
    """Pool bytes [n_pages, page_bytes] -> (K codes, K scales, V codes, V scales), each [n_pages, hkv, P, ...] views."""
    p = pages.view(pages.shape[0], hkv, -1)
    c, s = P * D // 2, P * D // 16
    cut = lambda a, b: p[..., a:b]  # noqa: E731
    half = c + s
    f16 = lambda t: t.contiguous().view(torch.float16).view(*t.shape[:2], P, D // 32)  # noqa: E731
    cod = lambda t: t.reshape(*t.shape[:2], P, D // 2)  # noqa: E731
    return (cod(cut(0, c)), f16(cut(c, half)), cod(cut(half, half + c)), f16(cut(half + c, 2 * half)))


def cached(pages, P, hkv, D, table_row, n):
    """float64 K and V [n, hkv, D] of a sequence of n tokens."""
    kc, ks, vc, vs = split_page(pages, P, hkv, D)
    ids = table_row[: -(-n // P)].long()
    out = []
    for c, s in ((kc, ks), (vc, vs)):
        x = unpack_head(c[ids], s[ids])                      # [pages, hkv, P, D]
        out.append(x.permute(0, 2, 1, 3).reshape(-1, hkv, D)[:n])
    return out


def quantise(x: torch.Tensor) -> torch.Tensor:
    """The values that 4 bits keep of float64 x [..., D]."""
    b = x.double().nan_to_num(0.0).clamp(-65504, 65504).unflatten(-1, (-1, 32))
    hi, lo = b.amax(-1, keepdim=True), b.amin(-1, keepdim=True)
    d = (torch.where(hi >= -lo, hi, lo) / -8).half().double()
    code = torch.floor(torch.where(d != 0, b / torch.where(d != 0, d, 1.0), 0.0) + 8.5).clamp(0, 15)
    return ((code - 8) * d).flatten(-2), d.expand_as(b).flatten(-2).abs()


def norm_rotate(x, w, cos, sin, pairs, eps):
    """x [T, heads, D], cos / sin [T, rot / 2] -> float64."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if cos is None:
        return x
    n = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = x.clone()
    if pairs:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = a * c - b * s, b * c + a * s
    return y


def attend(q, K, V, scale, causal=True, window=0, softcap=0.0):
    """One sequence: q [n, H, D], K and V [len, hkv, D] -> (out [n, H, D] in float64, bound factors).

    The second result bounds |error| of an implementation that rounds q, the values and the probabilities to 11-bit
    significands: each probability is then off by a relative 2^-11 + 2 dz, dz the largest error of a score, and by
    2^-25 where fp16 goes subnormal (a probability being held relative to a maximum that may lie 2^8 below the row's)."""
    n, H, D = q.shape
    L, hkv, _ = K.shape
    g = H // hkv
    out = torch.zeros(n, H, D, dtype=torch.float64)
    tol = torch.zeros(n, H, D, dtype=torch.float64)
    if L == 0:
        return out, tol
    q = q.double().view(n, hkv, g, D)
    z = torch.einsum("nhgd,jhd->nhgj", q, K) * scale
    dz = (torch.einsum("nhgd,jhd->nhgj", q.abs(), K.abs()) * abs(scale)).amax(-1) * 2.0 ** -11 + 1e-6
    if softcap > 0:
        z = softcap * torch.tanh(z / softcap)
        dz = dz + softcap * 2.0 ** -20
    pos = torch.arange(L - n, L)[:, None]
    j = torch.arange(L)[None]
    see = torch.ones(n, L, dtype=torch.bool)
    if causal:
        see = j <= pos
        if window:
            see &= j > pos - window
    z = z.masked_fill(~see[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    e = torch.where(see[:, None, None], torch.exp(z - torch.where(m.isfinite(), m, 0.0)), 0.0)
    l = e.sum(-1, keepdim=True)
    p = e / torch.where(l > 0, l, 1.0)
    o = torch.einsum("nhgj,jhd->nhgd", p, V)
    av = torch.einsum("nhgj,jhd->nhgd", p, V.abs())
    vmax = V.abs().amax()
    t = (2.0 ** -10 + 2 * dz[..., None] + 2.0 ** -17) * av + see.sum(-1)[:, None, None, None] * 2.0 ** -25 * vmax
    return o.reshape(n, H, D), t.reshape(n, H, D)
