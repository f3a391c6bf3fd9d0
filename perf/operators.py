"""Cases of the attention-side operators that stand in front of the lfm2moe FFN.

  norm    residual addition, RMSNorm and the Q8_K output (256 codes of 8 bits under one fp32 scale)
  append  per-head RMSNorm and position rotation of q and k, keys and values into a paged 4-bit cache
  attn    grouped-query attention over that cache, for single tokens, verify batches, prompts and chunks

Cache format (one pool per layer, uint8): page p is [kv head][K codes | K scales | V codes | V scales] for
`page` tokens.  A token's head is quantised in blocks of 32 values with an fp16 scale d: value = d * (code - 8),
d = m / -8 for the value m of largest magnitude (the positive one on a tie).  Codes lie in 64-wide spans of eight
32-bit words: nibble n of word w is value 32 * (n / 4) + 4 * w + n % 4 of the span.

Sequence b of a batch owns the q rows q_start[b] .. q_start[b + 1]; its cache holds kv_len[b] tokens with those
rows' tokens as the last ones; page_table[b][i] is the pool page of its tokens i * page ...
"""
import functools
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
SPAN = 64
NEG = float("-inf")


# ---- the cases ---------------------------------------------------------------------------------------------


def listed():
    return [
        # the decode batch of the 24-layer stack: 64 rows of D = 2048 before its MoE layer
        {"name": "norm_step", "op": "norm", "T": 64, "D": 2048, "delta": "bf16", "xb": False},
        # a prompt's rows, the fp32 output of the projection added
        {"name": "norm_prompt", "op": "norm", "T": 4096, "D": 2048, "delta": "f32", "xb": False},
        # an odd number of wide rows, with the normalised rows in 16 bits too (for a 16-bit projection)
        {"name": "norm_wide", "op": "norm", "T": 1021, "D": 5120, "delta": "bf16", "xb": True},
        # one token of each of 64 sequences enters the cache
        {"name": "append_step", "op": "append", "B": 64, "q": 1, "kv": 4096, "ragged": True, "H": 32, "Hkv": 8, "D": 64,
         "page": 64, "pairs": False, "rot": 64, "norm": True},
        # eight ragged prompts, pages of 16 tokens, a partial rotation of neighbouring values
        {"name": "append_prompts", "op": "append", "B": 8, "q": 1024, "kv": 1024, "ragged": True, "H": 32, "Hkv": 8,
         "D": 128, "page": 16, "pairs": True, "rot": 64, "norm": False},
        # one user's next token: latency counts
        {"name": "decode_one", "op": "attn", "B": 1, "q": 1, "kv": 1024, "ragged": False, "H": 32, "Hkv": 8, "D": 64,
         "page": 64, "causal": True, "window": 0, "cap": 0.0},
        # the 64-token decode step at ragged lengths up to 8192
        {"name": "decode_batch", "op": "attn", "B": 64, "q": 1, "kv": 8192, "ragged": True, "H": 32, "Hkv": 8, "D": 64,
         "page": 64, "causal": True, "window": 0, "cap": 0.0},
        # two very long contexts
        {"name": "decode_long", "op": "attn", "B": 2, "q": 1, "kv": 131072, "ragged": False, "H": 32, "Hkv": 8, "D": 128,
         "page": 128, "causal": True, "window": 0, "cap": 0.0},
        # speculative verification: 8 tokens of each of 16 sequences
        {"name": "verify", "op": "attn", "B": 16, "q": 8, "kv": 8192, "ragged": True, "H": 32, "Hkv": 8, "D": 64,
         "page": 64, "causal": True, "window": 0, "cap": 0.0},
        # a prompt of 4096 tokens from the beginning
        {"name": "prompt", "op": "attn", "B": 1, "q": 4096, "kv": 4096, "ragged": False, "H": 32, "Hkv": 8, "D": 64,
         "page": 64, "causal": True, "window": 0, "cap": 0.0},
        # a 2048-token chunk of a long prompt behind 14336 cached tokens
        {"name": "chunk", "op": "attn", "B": 1, "q": 2048, "kv": 16384, "ragged": False, "H": 32, "Hkv": 8, "D": 128,
         "page": 64, "causal": True, "window": 0, "cap": 0.0},
        # a mixed batch: ragged chunks behind ragged contexts, a sliding window, capped scores, five heads a group
        {"name": "mixed_window", "op": "attn", "B": 12, "q": 509, "kv": 6007, "ragged": True, "H": 20, "Hkv": 4, "D": 64,
         "page": 32, "causal": True, "window": 1024, "cap": 30.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attn", "attn", "attn"])
    if op == "norm":
        return {"op": op, "T": _log(rng, 1, 4096), "D": 256 * rng.choice([2, 3, 4, 5, 7, 8, 9, 10, 11, 13, 16, 20]), "delta": rng.choice(["bf16", "f32", "none"]),
                "xb": rng.random() < 0.4}
    hkv = rng.choice([1, 2, 4, 8])
    heads = {"H": hkv * rng.choice([1, 2, 3, 4, 4, 5, 8]), "Hkv": hkv, "D": rng.choice([64, 64, 128]),
             "page": rng.choice([16, 32, 64, 64, 128])}
    if op == "append":
        b = _log(rng, 1, 64)
        q = _log(rng, 1, max(1, 4096 // b))
        return {"op": op, "B": b, "q": q, "kv": q + _log(rng, 1, 4000) - 1, "ragged": rng.random() < 0.7, **heads,
                "pairs": rng.random() < 0.4, "rot": rng.choice([32, heads["D"], heads["D"]]), "norm": rng.random() < 0.5}
    kind = rng.choice(["one", "batch", "verify", "chunk"])
    if kind == "one":
        b, q, kv = rng.randint(1, 4), 1, _log(rng, 1, 131072)
    elif kind == "batch":
        b, q, kv = _log(rng, 5, 64), 1, _log(rng, 60, 8192)
    elif kind == "verify":
        b, q, kv = _log(rng, 1, 16), rng.randint(2, 16), _log(rng, 100, 8192)
    else:
        b, q = _log(rng, 1, 6), _log(rng, 17, 1500)
        kv = q + _log(rng, 1, 6000) - 1
    causal = rng.random() < 0.85
    return {"op": op, "B": b, "q": q, "kv": max(q, kv), "ragged": rng.random() < 0.7, **heads, "causal": causal,
            "window": rng.choice([0, 0, _log(rng, 1, 3000)]) if causal else 0, "cap": rng.choice([0.0, 0.0, 0.0, 20.0])}


# ---- lengths and bytes of a case ---------------------------------------------------------------------------


def lengths(case):
    """(q rows, cached tokens) of each sequence; a ragged batch spreads them between a quarter and the whole."""
    rows = []
    for b in range(case["B"]):
        u, v = ((b + 1) * 0.6180339887) % 1.0, ((b + 1) * 0.7548776662) % 1.0
        q = max(1, int(case["q"] * (0.25 + 0.75 * u))) if case["ragged"] else case["q"]
        kv = max(q, int(case["kv"] * (0.25 + 0.75 * v))) if case["ragged"] else case["kv"]
        rows.append((q, kv))
    return rows


def head_bytes(d):
    """Bytes of one token's key (or value) of one head: 4-bit codes and a 16-bit scale for 32 of them."""
    return d // 2 + d // 32 * 2


def visible(q, kv, causal, window):
    """(query, key) pairs that a head scores, and the cached tokens that some query sees."""
    if not causal:
        return q * kv, kv
    n = np.arange(kv - q + 1, kv + 1, dtype=np.int64)
    n = np.minimum(n, window) if window else n
    return int(n.sum()), int(min(kv, q - 1 + window)) if window else kv


def work(case):
    if case["op"] == "norm":
        n = case["T"] * case["D"]
        delta = {"none": 0, "bf16": 2, "f32": 4}[case["delta"]]
        return {"bytes": n * (4 + delta + 4 + (2 if case["xb"] else 0)) + n // 256 * 292 + 4 * case["D"], "flops": 8 * n}
    rows, d, h, hkv = lengths(case), case["D"], case["H"], case["Hkv"]
    t = sum(q for q, _ in rows)
    if case["op"] == "append":
        return {"bytes": t * (2 * h * d * 2 + 2 * hkv * d * 2 + 2 * hkv * head_bytes(d) + case["rot"] * 4), "flops": 8 * t * (h + 2 * hkv) * d}
    pairs = [visible(q, kv, case["causal"], case["window"]) for q, kv in rows]
    return {"bytes": sum(keys for _, keys in pairs) * hkv * 2 * head_bytes(d) + 2 * t * h * d * 2,
            "flops": 4 * d * h * sum(n for n, _ in pairs)}


# ---- the inputs --------------------------------------------------------------------------------------------


def quantise(x):
    """4-bit codes and scales of fp32 x [..., D]: (codes, fp16 scales)."""
    b = x.unflatten(-1, (-1, 32))
    hi, lo = b.amax(-1), b.amin(-1)
    m = torch.where(hi >= -lo, hi, lo).clamp(-65504.0, 65504.0)
    d = (m * -0.125).half()
    f = d.float()
    inv = torch.where(f != 0, 1.0 / f, torch.zeros_like(f))
    return torch.floor(b * inv.unsqueeze(-1) + 8.5).clamp(0, 15).flatten(-2), d


def values(codes, d):
    return ((codes.unflatten(-1, (-1, 32)) - 8.0) * d.float().unsqueeze(-1)).flatten(-2)


def pack(codes):
    """Codes [..., D] -> bytes [..., D / 2] in the cache's order."""
    n = codes.to(torch.uint8).unflatten(-1, (-1, 2, 8, 4)).transpose(-3, -2).flatten(-4)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def unpack(by):
    """Bytes [..., D / 2] -> fp32 codes [..., D]."""
    n = torch.stack((by & 15, by >> 4), -1).flatten(-2).unflatten(-1, (-1, 8, 2, 4))
    return n.transpose(-3, -2).flatten(-4).float()


def pool(n, case, gen, dev):
    """A layer's pool of n pages of keys and values as a model leaves them."""
    p, hkv, d = case["page"], case["Hkv"], case["D"]
    out = torch.empty(n, hkv, 2 * p * head_bytes(d), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 26) // (hkv * p * d))
    for at in range(0, n, step):
        m, o = min(step, n - at), 0
        for _ in range(2):
            c, s = quantise(torch.randn(m, hkv, p, d, generator=gen, device=dev))
            for part in (pack(c).flatten(-2), s.contiguous().view(torch.uint8).flatten(-2)):
                out[at : at + m, :, o : o + part.shape[-1]] = part
                o += part.shape[-1]
    return out.flatten(1)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(dev).manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    if case["op"] == "norm":
        t, d = case["T"], case["D"]
        s = {"x": rand(t, d) * 2, "delta": None, "w": 1 + 0.1 * rand(d)}
        if case["delta"] != "none":
            s["delta"] = rand(t, d).to(TYPES[case["delta"]])
        return {"case": case, **s}
    rows, p, h, hkv, d = lengths(case), case["page"], case["H"], case["Hkv"], case["D"]
    most = max(-(-kv // p) for _, kv in rows)
    total = sum(-(-kv // p) for _, kv in rows)
    order = torch.randperm(total + 3, generator=torch.Generator().manual_seed(int(seed))).tolist()
    table = torch.full((case["B"], most), -1, dtype=torch.int32)
    at = 0
    for b, (_, kv) in enumerate(rows):
        n = -(-kv // p)
        table[b, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
        at += n
    t = sum(q for q, _ in rows)
    starts = np.cumsum([0] + [q for q, _ in rows]).astype(np.int32)
    s = {"case": case, "n_pages": total + 3, "most_q": max(q for q, _ in rows), "most_kv": max(kv for _, kv in rows),
         "q_start": torch.from_numpy(starts).to(dev), "kv_len": torch.tensor([kv for _, kv in rows], dtype=torch.int32, device=dev),
         "table": table.to(dev)}
    if case["op"] == "append":
        ang = torch.arange(s["most_kv"], device=dev).float()[:, None] * 10000.0 ** (-torch.arange(0, case["rot"], 2, device=dev).float() / case["rot"])
        s |= {"cos": ang.cos(), "sin": ang.sin(), "q": rand(t, h, d).bfloat16(), "k": rand(t, hkv, d).bfloat16(), "v": rand(t, hkv, d).bfloat16(),
              "qn": 1 + 0.1 * rand(d) if case["norm"] else None, "kn": 1 + 0.1 * rand(d) if case["norm"] else None,
              "pages": torch.zeros(s["n_pages"], hkv * 2 * p * head_bytes(d), dtype=torch.uint8, device=dev)}
    else:
        s |= {"q": (1.5 * rand(t, h, d)).bfloat16(), "pages": pool(s["n_pages"], case, gen, dev), "scale": d ** -0.5}
    return s


# ---- one pass ----------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _norm, "append": _append, "attn": _attn}[state["case"]["op"]](state)


def _norm(s):
    x = s["x"] if s["delta"] is None else s["x"] + s["delta"].float()
    y = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * s["w"]
    b = y.unflatten(-1, (-1, 256))
    m = b.abs().amax(-1, keepdim=True)
    codes = torch.round(b * torch.where(m > 0, 127.0 / m, torch.zeros_like(m))).clamp(-128, 127)
    out = {"x": x, "q8": (codes * (m / 127.0)).flatten(-2).bfloat16()}
    return out | ({"xb": y.bfloat16()} if s["case"]["xb"] else {})


def _places(s):
    """(sequence, place among its rows, position in the cache) of each q row."""
    t = torch.arange(s["q"].shape[0], device=s["q"].device)
    b = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    i = t - s["q_start"].long()[b]
    return b, i, s["kv_len"].long()[b] - (s["q_start"][1:] - s["q_start"][:-1]).long()[b] + i


def _rotate(x, cos, sin, pairs):
    """x [T, heads, D] fp32, cos and sin [T, 1, rot / 2]: its first `rot` values turned, in neighbouring pairs or in halves."""
    n = cos.shape[-1]
    a, b = (x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]) if pairs else (x[..., :n], x[..., n : 2 * n])
    c, d = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((c, d), -1).flatten(-2) if pairs else torch.cat((c, d), -1)
    return torch.cat((y, x[..., 2 * n :]), -1)


def _append(s):
    case = s["case"]
    _, _, pos = _places(s)
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
    q, k = s["q"].float(), s["k"].float()
    if case["norm"]:
        q = q * (1.0 / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS)) * s["qn"]
        k = k * (1.0 / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS)) * s["kn"]
    q, k = _rotate(q, cos, sin, case["pairs"]), _rotate(k, cos, sin, case["pairs"])
    return {"q": q.bfloat16(), "k": values(*quantise(k)).bfloat16(), "v": values(*quantise(s["v"].float())).bfloat16()}


def _cached(s, which):
    """Keys (0) or values (1) of every sequence, [B, kv heads, tokens, D] fp32; what no token holds is zero."""
    case = s["case"]
    p, hkv, d = case["page"], case["Hkv"], case["D"]
    g = s["pages"].view(s["n_pages"], hkv, -1)[s["table"].long().clamp(min=0)]
    at = which * p * head_bytes(d)
    codes = unpack(g[..., at : at + p * d // 2].unflatten(-1, (p, d // 2)))
    d16 = g[..., at + p * d // 2 : at + p * head_bytes(d)].contiguous().view(torch.float16).unflatten(-1, (p, d // 32))
    x = values(codes, d16).transpose(1, 2).flatten(2, 3)
    held = torch.arange(x.shape[2], device=x.device) < s["kv_len"][:, None]
    return torch.where(held[:, None, :, None], x, torch.zeros_like(x))


def _attn(s):
    case = s["case"]
    h, hkv, d = case["H"], case["Hkv"], case["D"]
    b, i, _ = _places(s)
    k, v = _cached(s, 0), _cached(s, 1)
    n, keys, g = s["most_q"], k.shape[2], h // hkv
    q = torch.zeros(case["B"], n, h, d, device=k.device)
    q[b, i] = s["q"].float()
    q = q.view(case["B"], n, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(case["B"], hkv, g * n, d)
    z = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    if case["cap"]:
        z = torch.tanh(z / case["cap"]) * case["cap"]
    rows = s["q_start"][1:] - s["q_start"][:-1]
    pos = (s["kv_len"] - rows)[:, None, None] + torch.arange(n, device=k.device)[:, None]
    j = torch.arange(keys, device=k.device)
    see = (j < s["kv_len"][:, None, None]).expand(-1, n, -1)
    if case["causal"]:
        see = see & (j <= pos)
        if case["window"]:
            see = see & (j > pos - case["window"])
    z = torch.where(see[:, None, None], z.unflatten(2, (g, n)), NEG).flatten(2, 3)
    m = z.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(z - m)
    den = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(den > 0, den, torch.ones_like(den))
    o = o.view(case["B"], hkv, g, n, d).permute(0, 3, 1, 2, 4).reshape(case["B"], n, h, d)
    return {"out": o[b, i].to(s["q"].dtype)}


@functools.lru_cache(maxsize=None)
def _library():
    """The handle of the device, which a program makes once."""
    from laii_b200.attn import GpuAttn
    from laii_b200.moe import GpuMoE

    return GpuAttn(GpuMoE(torch.cuda.current_device()))


def _plan(s):
    """What a program keeps beside its buffers: the descriptions of the cache, of the batch and of the rotation."""
    from laii_b200.attn import KVBatch, KVPages, Rope

    case = s["case"]
    cache = KVPages(s["pages"], page_tokens=case["page"], n_kv_heads=case["Hkv"], head_dim=case["D"])
    batch = KVBatch(s["q_start"], s["kv_len"], s["table"], max_kv_len=s["most_kv"])
    if case["op"] == "attn":
        return cache, batch, None
    return cache, batch, Rope(s["cos"], s["sin"], pairs=case["pairs"], q_norm=s["qn"], k_norm=s["kn"], eps=EPS)


def _run_own(s):
    lib, case = _library(), s["case"]
    if case["op"] == "norm":
        x, xb, q8 = lib.add_rmsnorm(s["x"], s["delta"], s["w"], eps=EPS, xb_dtype=torch.bfloat16 if case["xb"] else None)
        out = {"x": x, "q8": lib.read_q8(q8, torch.bfloat16)}
        return out | ({"xb": xb} if case["xb"] else {})
    if "plan" not in s:
        s["plan"] = _plan(s)
    cache, batch, rope = s["plan"]
    if case["op"] == "append":
        q = lib.append(cache, batch, s["q"], s["k"], s["v"], rope)
        k, v = lib.read(cache, batch, n_tokens=q.shape[0], dtype=torch.bfloat16)
        return {"q": q, "k": k, "v": v}
    return {"out": lib.attend(cache, batch, s["q"], scale=s["scale"], causal=case["causal"], window=case["window"], softcap=case["cap"])}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attn": _exact_attn}[case["op"]](s)


def _exact_norm(s):
    x = s["x"].double() + (0 if s["delta"] is None else s["delta"].double())
    y = x / (x.pow(2).sum(1, keepdim=True) / x.shape[1] + EPS).sqrt() * s["w"].double()
    blocks = y.reshape(x.shape[0], -1, 256)
    d = blocks.abs().max(2, keepdim=True).values / 127
    out = {"x": x, "q8": (torch.round(blocks / d.clamp(min=1e-300)) * d).reshape(x.shape)}
    return out | ({"xb": y} if s["case"]["xb"] else {})


def _exact_quantised(x):
    """The 4-bit values nearest below or at the half step of x [..., D] in 64 bits; the scale is held in 16."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    at = b.abs().max(-1).values
    m = torch.where((b == at[..., None]).any(-1), at, -at)
    d = (m / -8).half().double()[..., None]
    return (((b / d + 0.5).floor()).clamp(-8, 7) * d).reshape(x.shape)


def _exact_append(s):
    case = s["case"]
    rows, n = lengths(case), case["rot"] // 2
    pos = torch.cat([torch.arange(kv - q, kv) for q, kv in rows]).to(s["q"].device)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    out = {}
    for name, w in (("q", s["qn"]), ("k", s["kn"])):
        x = s[name].double()
        if case["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
        first, second = (list(range(0, 2 * n, 2)), list(range(1, 2 * n, 2))) if case["pairs"] else (list(range(n)), list(range(n, 2 * n)))
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        out[name] = y
    return {"q": out["q"], "k": _exact_quantised(out["k"]), "v": _exact_quantised(s["v"].double())}


def _exact_attn(s):
    case = s["case"]
    h, hkv, d, p = case["H"], case["Hkv"], case["D"], case["page"]
    if work(case)["flops"] > 1.5e12:
        return None
    dev, g, out, at = s["q"].device, h // hkv, [], 0
    # value i of a head: its byte and shift in the token's codes
    i = np.arange(d)
    nib = (i % SPAN) // 4 % 8 * 8 + (i % SPAN) // 32 * 4 + i % 4
    byte = torch.from_numpy(i // SPAN * 32 + nib // 2).to(dev)
    shift = torch.from_numpy(nib % 2 * 4).to(dev)
    block = torch.from_numpy(i // 32).to(dev)
    pages = s["pages"].view(s["n_pages"], hkv, 2, p * head_bytes(d))
    for b, (n, kv) in enumerate(lengths(case)):
        held = pages[s["table"][b, : -(-kv // p)].long()]
        q = s["q"][at : at + n].double().view(n, hkv, g, d)
        at += n
        o = torch.empty(n, hkv, g, d, dtype=torch.float64, device=dev)
        first = max(0, kv - n - case["window"] + 1) if case["causal"] and case["window"] else 0
        for head in range(hkv):
            kvv = []
            for which in (0, 1):
                raw = held[:, head, which]
                codes = raw[:, : p * d // 2].reshape(-1, d // 2)[first:kv]
                scales = raw[:, p * d // 2 :].contiguous().view(torch.float16).reshape(-1, d // 32)[first:kv].double()
                kvv.append((((codes[:, byte].int() >> shift) & 15).double() - 8) * scales[:, block])
            k, v = kvv
            step = max(1, (1 << 27) // max(1, g * k.shape[0]))
            for a in range(0, n, step):
                z = torch.einsum("nhd,jd->nhj", q[a : a + step, head], k) * s["scale"]
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                if case["causal"]:
                    pos = torch.arange(kv - n, kv, device=dev)[a : a + step, None]
                    j = torch.arange(first, kv, device=dev)
                    hide = (j > pos) | ((j <= pos - case["window"]) if case["window"] else (j < 0))
                    z = z.masked_fill(hide[:, None], NEG)
                o[a : a + step, head] = torch.einsum("nhj,jd->nhd", torch.softmax(z, -1), v)
        out.append(o.reshape(n, h, d))
    return {"out": torch.cat(out)}
