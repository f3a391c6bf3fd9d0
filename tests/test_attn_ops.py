"""The attention-side operators on the GPU against their definitions in 64 bits (tests/attn_ref.py)."""
import ctypes
import math

import pytest
import torch

import attn_ref as ref

pytestmark = pytest.mark.gpu

EPS = 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# unit roundoff: the largest relative error of rounding to nearest at 24, 11 and 8 significant bits
ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def lib():
    from laii_b200.attn import GpuAttn
    from laii_b200.moe import GpuMoE
    with GpuMoE(0) as moe:
        yield GpuAttn(moe)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def dev(t, dtype=None):
    return None if t is None else t.to("cuda", dtype)


# ---- residual addition, RMSNorm, Q8_K ---------------------------------------------------------------------------


@pytest.mark.parametrize("D", [256, 768, 2048, 8192])
@pytest.mark.parametrize("T,delta,xb,inplace", [(1, "bf16", None, False), (3, "f32", "f32", True), (65, None, "bf16", False),
                                                (130, "f16", "f16", True)])
def test_add_rmsnorm(lib, D, T, delta, xb, inplace):
    g = gen(D + T)
    x = torch.randn(T, D, generator=g) * 3
    d = None if delta is None else torch.randn(T, D, generator=g).to(DTYPES[delta])
    w = 1 + 0.2 * torch.randn(D, generator=g)
    x[0, : min(D, 256)] *= 1e-3  # a quiet block beside loud ones
    xd = dev(x)
    xo, xbo, q8 = lib.add_rmsnorm(xd, dev(d), dev(w), EPS, x_out=xd if inplace else None,
                                  xb_dtype=None if xb is None else DTYPES[xb])
    lib.moe.sync()
    y32 = x + (0 if d is None else d.float())           # one fp32 addition: exactly this
    assert torch.equal(xo.cpu(), y32)
    y = y32.double()
    n = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * w.double()
    # the sum of squares in fp32 (at most 8 + 5 + 32 additions deep), one root, two divisions, two products
    tol = 64 * 2.0 ** -24
    if xb is not None:
        assert ((xbo.cpu().double() - n).abs() <= (tol + ULP[xb]) * n.abs() + (2.0 ** -25 if xb == "f16" else 1e-38)).all()
    raw = q8.cpu()
    s = raw[..., :4].contiguous().view(torch.float32).double()          # [T, nb, 1]
    codes = raw[..., 4:260].contiguous().view(torch.int8).double()
    sums = raw[..., 260:].contiguous().view(torch.int16).long()
    blocks = n.view(T, -1, 256)
    m = blocks.abs().amax(-1, keepdim=True)
    assert ((s - m / 127).abs() <= (tol + 2.0 ** -23) * m / 127).all()
    assert ((codes * s - blocks).abs() <= s * (0.5 + 256 * tol)).all()  # nearest code
    assert torch.equal(sums, codes.long().view(T, -1, 16, 16).sum(-1))
    for name, dt in DTYPES.items():
        v = lib.read_q8(q8, dt).cpu()
        assert torch.equal(v, (codes.float() * s.float()).view(T, D).to(dt)), name


def test_add_rmsnorm_zero_rows_and_parts(lib):
    x = torch.zeros(2, 512, device="cuda")
    xo, xb, q8 = lib.add_rmsnorm(x, None, None, EPS, xb_dtype=torch.float32)
    assert not xo.any() and not xb.any() and not q8.any()
    xo, xb, q8 = lib.add_rmsnorm(x, None, None, EPS, q8=False)
    assert xb is None and q8 is None
    assert lib.add_rmsnorm(x[:0], None, None, EPS)[0].shape == (0, 512)
    assert lib.read_q8(torch.empty(0, 2, 292, dtype=torch.uint8, device="cuda"), torch.float32).shape == (0, 512)


def test_add_rmsnorm_without_a_residual_output(lib):
    """The C entry takes NULL for any output but not for all of them."""
    x = torch.randn(4, 256, generator=gen(1)).cuda()
    q8 = torch.empty(4, 1, 292, dtype=torch.uint8, device="cuda")
    a = (lib.moe._h, x.data_ptr(), None, 0, 4, 256, None, EPS, None, None, 0)
    assert lib._lib.lfm_gpu_add_rmsnorm(*a, q8.data_ptr(), lib._stream()) == 0
    assert torch.equal(q8, lib.add_rmsnorm(x, None, None, EPS)[2])
    assert lib._lib.lfm_gpu_add_rmsnorm(*a, None, None) == -1


def test_add_rmsnorm_matches_the_layer_router(lib):
    """The Q8_K rows are those of the MoE layer's own norm, but for codes at a rounding boundary."""
    from laii_b200 import synth
    L = synth.make_moe_layer(512, 8, 2, 512, layer=0)
    x = synth.make_hidden(5, 512, seed_offset=3)
    lib.moe.upload_layer(0, L)
    _, _, q = lib.moe.debug_route(0, x)
    want = torch.from_numpy(q.reshape(5, 2, 292))
    _, _, got = lib.add_rmsnorm(torch.from_numpy(x).cuda(), None, torch.from_numpy(L.ffn_norm).cuda(), L.eps)
    a, b = (t[..., 4:260].contiguous().view(torch.int8).int() for t in (want, got.cpu()))
    assert (a - b).abs().max() <= 1 and (a != b).float().mean() < 1e-3


@pytest.mark.parametrize("change,status", [
    (dict(D=255), -2), (dict(D=8448), -2), (dict(dt=12), -2), (dict(eps=-1.0), -1), (dict(eps=math.nan), -1),
    (dict(x=None), -1), (dict(x=4), -1), (dict(q8=2), -1)])
def test_add_rmsnorm_refusals(lib, change, status):
    x = torch.zeros(4, 512, device="cuda")
    p = x.data_ptr()
    a = {"x": p, "dt": 0, "D": 256, "eps": EPS, "q8": p} | {
        k: (p + v if k in ("x", "q8") and v else v) for k, v in change.items()}
    st = lib._lib.lfm_gpu_add_rmsnorm(lib.moe._h, a["x"], p, a["dt"], 2, a["D"], None, a["eps"], p, None, 0, a["q8"], None)
    assert st == status
    lib.moe.sync()


# ---- a batch with its cache -------------------------------------------------------------------------------------


class Case:
    """A ragged batch with a scattered page table; unused pool bytes are 0xFF (NaN scales), unused entries -1."""

    def __init__(self, rows, P, hkv, D, seed=0, fill=True, spare=3, scale=1.0):
        from laii_b200.attn import KVBatch, KVPages
        self.rows, self.P, self.hkv, self.D = rows, P, hkv, D
        self.T = sum(q for q, _ in rows)
        need = [-(-n // P) for _, n in rows]
        order = torch.randperm(sum(need) + spare, generator=gen(seed)).int()
        self.table = torch.full((max(1, len(rows)), max([1] + need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.pages = torch.full((sum(need) + spare, hkv * 2 * P * (D // 2 + D // 16)), 255, dtype=torch.uint8)
        if fill:
            kc, ks, vc, vs = ref.split_page(self.pages, P, hkv, D)
            raw = self.pages.view(self.pages.shape[0], hkv, -1)
            c, s, half = P * D // 2, P * D // 16, P * (D // 2 + D // 16)
            g = gen(seed + 1)
            for b, (_, n) in enumerate(rows):
                for i in range(need[b]):
                    m = min(P, n - i * P)
                    for o in (0, half):
                        page = raw[int(self.table[b, i])]
                        page[:, o:o + m * D // 2] = torch.randint(0, 256, (hkv, m * D // 2), generator=g, dtype=torch.uint8)
                        sc = (scale * (0.1 + 0.3 * torch.rand(hkv, m * D // 32, generator=g))).half()
                        sc *= (torch.randint(0, 2, sc.shape, generator=g) * 2 - 1)
                        page[:, o + c:o + c + m * D // 16] = sc.view(torch.uint8).view(hkv, -1)
        starts = [0]
        for q, _ in rows:
            starts.append(starts[-1] + q)
        self.starts = starts
        self.cache = KVPages(self.pages.cuda(), P, hkv, D)
        self.batch = KVBatch(torch.tensor(starts, dtype=torch.int32).cuda(),
                             torch.tensor([n for _, n in rows], dtype=torch.int32).cuda(), self.table.cuda(),
                             max([n for _, n in rows], default=0))

    def kv(self, b):
        return ref.cached(self.pages, self.P, self.hkv, self.D, self.table[b], self.rows[b][1])


def check_attend(c, q, out, name, scale, **kw):
    for b, (n, _) in enumerate(c.rows):
        a = slice(c.starts[b], c.starts[b] + n)
        K, V = c.kv(b)
        want, tol = ref.attend(q[a].cpu(), K, V, scale, **kw)
        got = out[a].cpu().double()
        assert torch.isfinite(got).all()
        err = (got - want).abs()
        bound = tol + ULP[name] * want.abs() + (2.0 ** -25 if name == "f16" else 0) + 1e-30
        assert (err <= bound).all(), (b, float((err / bound).max()))


ROWS = {
    "one": [(1, 1)],
    "decode": [(1, 5), (1, 64), (1, 129), (1, 333), (1, 16)],
    "empty": [(0, 0), (2, 0), (1, 40), (0, 17), (3, 1)],
    "verify": [(8, 100), (3, 3), (5, 261)],
    "prompt": [(130, 130), (1, 1), (67, 200), (300, 300)],
}


@pytest.mark.parametrize("kind", list(ROWS))
@pytest.mark.parametrize("P,hkv,G,D,name", [(16, 2, 4, 64, "bf16"), (64, 1, 1, 64, "f32"), (128, 2, 3, 128, "f16"),
                                            (32, 1, 8, 128, "bf16"), (64, 1, 16, 64, "bf16"), (16, 1, 40, 128, "f16")])
def test_attend(lib, kind, P, hkv, G, D, name):
    c = Case(ROWS[kind], P, hkv, D, seed=D + P)
    q = (torch.randn(c.T, hkv * G, D, generator=gen(7)) * 0.5).to(DTYPES[name])
    out = lib.attend(c.cache, c.batch, q.cuda())
    lib.moe.sync()
    check_attend(c, q, out, name, D ** -0.5)
    assert torch.equal(out, lib.attend(c.cache, c.batch, q.cuda()))  # the same bits again


@pytest.mark.parametrize("kind", ["decode", "verify", "prompt"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=1), dict(window=33), dict(window=100000), dict(softcap=2.0),
                                dict(softcap=30.0, window=70), dict(causal=False, softcap=5.0)])
def test_attend_masks_and_caps(lib, kind, D, kw):
    c = Case(ROWS[kind], 32, 2, D, seed=D)
    q = (torch.randn(c.T, 8, D, generator=gen(9))).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda(), scale=0.11, **kw)
    lib.moe.sync()
    check_attend(c, q, out, "bf16", 0.11, **kw)


@pytest.mark.parametrize("rows", [[(1, 5000), (1, 1), (2, 2500)], [(40, 3000), (1, 700)], [(200, 2100)], [(17, 4099)]])
@pytest.mark.parametrize("D,G", [(64, 4), (128, 5)])
def test_attend_long(lib, rows, D, G):
    c = Case(rows, 64, 1, D, seed=5)
    q = (torch.randn(c.T, G, D, generator=gen(2)) * 0.7).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda())
    lib.moe.sync()
    check_attend(c, q, out, "bf16", D ** -0.5)


@pytest.mark.parametrize("rows", [[(1, 900)], [(80, 900)]])
def test_attend_growing_scores(lib, rows):
    """The running maximum moves many times, by much, in both directions; large and tiny scales."""
    for scale in (4.0, -4.0, 1e-4, 0.0):
        c = Case(rows, 16, 1, 64, seed=11)
        q = torch.randn(c.T, 4, 64, generator=gen(4)).bfloat16()
        out = lib.attend(c.cache, c.batch, q.cuda(), scale=scale)
        lib.moe.sync()
        check_attend(c, q, out, "bf16", scale)


@pytest.mark.parametrize("scale", [300.0, 2.0 ** -9])
def test_attend_cache_of_large_and_small_values(lib, scale):
    c = Case([(1, 200), (90, 150)], 16, 1, 64, seed=3, scale=scale)
    q = (torch.randn(c.T, 4, 64, generator=gen(4)) / scale).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda())
    lib.moe.sync()
    check_attend(c, q, out, "bf16", 0.125)


@pytest.mark.parametrize("rows", [[(1, 70), (1, 200)], [(140, 200), (70, 70)]])
def test_attend_padding_strides_streams_and_hints(lib, rows):
    """Rows of a fused projection, rows that no sequence owns, another stream, any length hint."""
    c = Case(rows, 64, 2, 64, seed=1)
    fused = torch.randn(c.T + 3, 12, 64, generator=gen(3)).bfloat16().cuda()
    q = fused[:, 2:10]
    out = torch.full((c.T + 3, 10, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lib.attend(c.cache, c.batch, q, out=out[:, 1:9])
    s.synchronize()
    lib.moe.sync()
    check_attend(c, q, out[:, 1:9], "bf16", 0.125)
    assert (out[c.T:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 9] == 7).all()
    for hint in (1, 0, 100000):
        c.batch._c.max_kv_len = hint
        o = lib.attend(c.cache, c.batch, q)
        check_attend(c, q, o, "bf16", 0.125)


def test_attend_two_streams_share_the_scratch(lib):
    """Long sequences joined from parts, from two streams in turn."""
    c = Case([(1, 20000)], 64, 1, 64, seed=6)
    q = torch.randn(1, 4, 64, generator=gen(8)).bfloat16().cuda()
    q2 = torch.randn(1, 4, 64, generator=gen(9)).bfloat16().cuda()
    want, want2 = lib.attend(c.cache, c.batch, q), lib.attend(c.cache, c.batch, q2)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        for s, x in ((a, q), (b, q2)):
            with torch.cuda.stream(s):
                outs.append(lib.attend(c.cache, c.batch, x))
    torch.cuda.synchronize()
    lib.moe.sync()
    assert all(torch.equal(o, want if i % 2 == 0 else want2) for i, o in enumerate(outs))


def test_attend_in_a_graph_follows_the_lengths(lib):
    """A captured call reads lengths, tables and rows anew at every replay."""
    c = Case([(1, 700), (1, 90)], 16, 1, 64, seed=2)
    q = torch.randn(2, 4, 64, generator=gen(1)).bfloat16().cuda()
    out = torch.empty_like(q)
    lib.reserve()
    lib.attend(c.cache, c.batch, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lib.attend(c.cache, c.batch, q, out=out)
    for n in (700, 33, 512, 1):
        c.rows[0] = (1, n)
        c.batch._keep[1].copy_(torch.tensor([n, 90], dtype=torch.int32))
        q.copy_(torch.randn(2, 4, 64, generator=gen(n)).bfloat16())
        g.replay()
        torch.cuda.synchronize()
        check_attend(c, q, out, "bf16", 0.125)
    lib.moe.sync()


def test_attend_offsets_beyond_32_bits(lib):
    """A pool of more than 2^32 bytes, the sequence's pages at its end."""
    from laii_b200.attn import KVPages
    c = Case([(3, 300), (70, 150)], 128, 2, 128, seed=4)
    per = c.pages.shape[1]
    n = (1 << 32) // per + 40
    big = torch.empty(n, per, dtype=torch.uint8, device="cuda")
    shift = n - c.pages.shape[0]
    big[shift:].copy_(c.pages)
    table = torch.where(c.table >= 0, c.table + shift, c.table)
    c.batch._keep[2].copy_(table)
    q = torch.randn(c.T, 8, 128, generator=gen(6)).bfloat16()
    out = lib.attend(KVPages(big, 128, 2, 128), c.batch, q.cuda())
    lib.moe.sync()
    check_attend(c, q, out, "bf16", 128 ** -0.5)
    k, _ = lib.read(KVPages(big, 128, 2, 128), c.batch, c.T, torch.float32)
    assert torch.equal(k[:3].cpu().double(), c.kv(0)[0][-3:])


@pytest.mark.parametrize("rows", [[(1, 100), (1, 100)], [(90, 100), (1, 100)]])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_attend_bad_page_is_reported(lib, rows, bad):
    from laii_b200.moe import MoEError
    c = Case(rows, 16, 1, 64, seed=4)
    t = c.table.clone()
    t[1, 3] = bad
    c.batch._keep[2].copy_(t)
    q = torch.randn(c.T, 4, 64, generator=gen(6)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda())
    with pytest.raises(MoEError) as e:
        lib.moe.sync()
    assert e.value.status == -10
    c.rows = rows[:1]
    check_attend(c, q, out, "bf16", 0.125)  # the other sequence is right
    lib.moe.sync()


@pytest.mark.parametrize("rows", [[(1, 100)], [(90, 100)]])
def test_attend_table_too_short_is_reported(lib, rows):
    from laii_b200.moe import MoEError
    c = Case(rows, 16, 1, 64, seed=4)
    c.batch._keep[1].copy_(torch.tensor([1000], dtype=torch.int32))
    lib.attend(c.cache, c.batch, torch.randn(c.T, 4, 64).bfloat16().cuda())
    with pytest.raises(MoEError) as e:
        lib.moe.sync()
    assert e.value.status == -10
    lib.moe.sync()


@pytest.mark.parametrize("rows,q_start,kv_len", [([(1, 50), (1, 50)], [0, 5, 1], [50, 50]), ([(1, 50), (1, 50)], [-3, 1, 2], [50, 50]),
                                                 ([(1, 50), (1, 50)], [0, 1, 900], [50, 50]), ([(1, 50), (1, 50)], [0, 1, 2], [-5, 50]),
                                                 ([(100, 150), (1, 50)], [0, 2 ** 31 - 1, -2 ** 31], [150, 50]),
                                                 ([(100, 150), (1, 50)], [0, 100, 101], [-2 ** 31, 50])])
def test_attend_nonsense_offsets_stay_in_bounds(lib, rows, q_start, kv_len):
    """Offsets and lengths that describe no batch: whatever is computed, nothing outside the rows is touched."""
    from laii_b200.moe import MoEError
    c = Case(rows, 16, 1, 64, seed=4)
    c.batch._keep[0].copy_(torch.tensor(q_start, dtype=torch.int32))
    c.batch._keep[1].copy_(torch.tensor(kv_len, dtype=torch.int32))
    buf = torch.full((c.T + 2, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    lib.attend(c.cache, c.batch, torch.randn(c.T, 4, 64).bfloat16().cuda(), out=buf[1:-1])
    try:
        lib.moe.sync()
    except MoEError as e:
        assert e.status == -10
    assert (buf[0] == 5).all() and (buf[-1] == 5).all()
    lib.moe.sync()


def _kv(lib, **change):
    from laii_b200 import _native
    c = Case([(2, 20)], 16, 2, 64)
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device="cuda")
    c.batch.rows(2)
    kv, bt = c.cache._c, c.batch._c
    a = {"n_heads": 4, "scale": 0.1, "causal": 1, "window": 0, "cap": 0.0, "type": 30, "q": q.data_ptr(), "qs": 256,
         "out": q.data_ptr(), "os": 256} | {k: v for k, v in change.items() if not k.startswith(("kv_", "bt_"))}
    for k, v in change.items():
        if k.startswith("kv_"):
            setattr(kv, k[3:], v)
        if k.startswith("bt_"):
            setattr(bt, k[3:], v)
    if "qoff" in change:
        a["q"] += change["qoff"]
    st = lib._lib.lfm_gpu_attn_forward(lib.moe._h, ctypes.byref(kv), ctypes.byref(bt), a["n_heads"], a["scale"], a["causal"],
                                       a["window"], a["cap"], a["type"], a["q"], a["qs"], a["out"], a["os"], None)
    text = lib._lib.lfm_gpu_moe_last_error(lib.moe._h)
    assert _native is not None
    return st, text


@pytest.mark.parametrize("change,status", [
    ({}, 0), (dict(n_heads=3), -1), (dict(n_heads=0), -1), (dict(scale=math.inf), -1), (dict(scale=math.nan), -1),
    (dict(window=3, causal=0), -1), (dict(cap=-1.0), -1), (dict(cap=math.nan), -1), (dict(type=12), -2), (dict(q=None), -1),
    (dict(out=None), -1), (dict(qoff=2), -1), (dict(qs=255), -1), (dict(qs=128), -1), (dict(os=260), -1),
    (dict(kv_head_dim=96), -2), (dict(kv_page_tokens=48), -2), (dict(kv_n_kv_heads=0), -2), (dict(kv_pages=None), -1),
    (dict(kv_n_pages=0), -1), (dict(bt_q_start=None), -1), (dict(bt_kv_len=None), -1), (dict(bt_page_table=None), -1),
    (dict(bt_table_stride=0), -1), (dict(bt_table_stride=2 ** 28), -1), (dict(bt_n_seqs=2 ** 21), -1),
    (dict(bt_n_tokens=2 ** 25), -1), (dict(bt_n_tokens=0), 0), (dict(bt_n_seqs=0), 0)])
def test_attend_refusals(lib, change, status):
    st, text = _kv(lib, **change)
    assert st == status, text
    lib.moe.sync()


def test_python_refusals(lib):
    from laii_b200.attn import KVBatch, KVPages, Rope
    c = Case([(2, 20)], 16, 2, 64)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (q.double(), q.cpu(), q[:, :, :32], q.transpose(0, 1), q.reshape(2, 256)):
        with pytest.raises(ValueError):
            lib.attend(c.cache, c.batch, bad)
    with pytest.raises(ValueError):
        lib.attend(c.cache, c.batch, q, out=q.float())
    with pytest.raises(ValueError):
        lib.append(c.cache, c.batch, q, q[:, :2], None)
    with pytest.raises(ValueError):
        lib.append(c.cache, c.batch, q, q[:, :2], q[:1, :2])
    with pytest.raises(ValueError):
        KVPages(c.cache.pages[:, :-1], 16, 2, 64)
    with pytest.raises(ValueError):
        KVBatch(c.batch._keep[0].long(), c.batch._keep[1], c.batch._keep[2])
    with pytest.raises(ValueError):
        lib.append(c.cache, c.batch, q, None, None, Rope(q_norm=torch.ones(32, device="cuda")))
    with pytest.raises(ValueError):
        lib.add_rmsnorm(torch.zeros(2, 256, device="cuda").T, None, None)


# ---- keys and values into the cache -------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", list(ROWS))
@pytest.mark.parametrize("P,hkv,G,D,name,rot,pairs,norm", [
    (16, 2, 4, 64, "bf16", 64, False, True), (64, 1, 1, 64, "f32", 32, True, False), (128, 3, 3, 128, "f16", 128, False, True),
    (32, 1, 8, 128, "bf16", 48, False, False), (64, 5, 2, 64, "bf16", 0, False, True), (16, 2, 1, 128, "f32", 128, True, True)])
def test_append(lib, kind, P, hkv, G, D, name, rot, pairs, norm):
    from laii_b200.attn import Rope
    c = Case(ROWS[kind], P, hkv, D, seed=P, fill=False)
    g = gen(D + rot)
    fused = torch.randn(c.T + 1, hkv * (G + 2), D, generator=g).to(DTYPES[name])
    q, k, v = fused[:, :hkv * G], fused[:, hkv * G:hkv * (G + 1)], fused[:, hkv * (G + 1):]
    n_pos = max(n for _, n in c.rows) + 1
    ang = torch.rand(n_pos, rot // 2, generator=g) * 6.28
    cos, sin = (ang.cos(), ang.sin()) if rot else (None, None)
    qn, kn = (1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)) if norm else (None, None)
    rope = Rope(dev(cos), dev(sin), pairs=pairs, q_norm=dev(qn), k_norm=dev(kn), eps=EPS)
    fd = fused.cuda()
    qo = torch.full((c.T + 1, hkv * G, D), 3.0, dtype=DTYPES[name], device="cuda")
    before = c.cache.pages.clone()
    # rows whose position would be negative are refused on the device and reported
    bad = any(n < m for m, n in c.rows)
    lib.append(c.cache, c.batch, fd[:, :hkv * G], fd[:, hkv * G:hkv * (G + 1)], fd[:, hkv * (G + 1):], rope, q_out=qo)
    if bad:
        from laii_b200.moe import MoEError
        with pytest.raises(MoEError):
            lib.moe.sync()
    lib.moe.sync()
    assert (qo[c.T:] == 3).all()
    after = c.cache.pages.cpu()
    touched = torch.zeros_like(before.cpu(), dtype=torch.bool)
    kb, sb, half = P * D // 2, P * D // 16, P * (D // 2 + D // 16)
    mark = touched.view(touched.shape[0], hkv, 2, half)
    parts = ref.split_page(after, P, hkv, D)
    tol = 64 * 2.0 ** -24
    for b, (m, n) in enumerate(c.rows):
        for i in range(m):
            t, pos = c.starts[b] + i, n - m + i
            if pos < 0:
                continue
            ct, st = (cos[pos:pos + 1], sin[pos:pos + 1]) if rot else (None, None)
            wq = ref.norm_rotate(q[t:t + 1], qn, ct, st, pairs, EPS)
            size = wq.abs().amax()
            assert ((qo[t].cpu().double() - wq[0]).abs() <= ULP[name] * wq[0].abs() + tol * size + 2.0 ** -25).all()
            page, slot = int(c.table[b, pos // P]), pos % P
            mark[page, :, :, slot * D // 2:(slot + 1) * D // 2] = True
            mark[page, :, :, kb + slot * D // 16:kb + (slot + 1) * D // 16] = True
            for x, (cc, ss) in ((ref.norm_rotate(k[t:t + 1], kn, ct, st, pairs, EPS)[0], parts[:2]), (v[t].double(), parts[2:])):
                got = ref.unpack_head(cc[page, :, slot], ss[page, :, slot])
                want, d = ref.quantise(x)
                # the same code, or the neighbour where the value lies within rounding of the boundary; the scale
                # within a unit of fp16
                near = (got - want).abs() <= 8 * 2.0 ** -10 * d + 2.0 ** -23
                edge = ((x / torch.where(d > 0, d, 1.0) - torch.floor(x / torch.where(d > 0, d, 1.0))) - 0.5).abs() < 1e-3
                assert (near | (edge & ((got - want).abs() <= 1.01 * d))).all()
                assert ((got - x).abs() <= 1.01 * d).all()
    assert torch.equal(after[~touched], before.cpu()[~touched])
    kr, vr = lib.read(c.cache, c.batch, c.T, torch.float32)
    if bad:
        with pytest.raises(Exception):
            lib.moe.sync()
    lib.moe.sync()
    for b, (m, n) in enumerate(c.rows):
        for i in range(max(0, m - n), m):
            t, pos = c.starts[b] + i, n - m + i
            page, slot = int(c.table[b, pos // P]), pos % P
            assert torch.equal(kr[t].cpu().double(), ref.unpack_head(parts[0][page, :, slot], parts[1][page, :, slot]))
            assert torch.equal(vr[t].cpu().double(), ref.unpack_head(parts[2][page, :, slot], parts[3][page, :, slot]))


def test_append_exact_codes(lib):
    """Without a norm the arithmetic is that of the definition in fp32, bit for bit: extremes of both signs, ties,
    zeros, values that leave fp16, infinities and NaN."""
    c = Case([(6, 6)], 16, 1, 64, fill=False)
    v = torch.randn(6, 1, 64, generator=gen(5))
    v[1, 0, :32] = 0
    v[2, 0, 0], v[2, 0, 1] = 4.0, -4.0            # a tie: the positive one
    v[2, 0, 2:32] = torch.linspace(-3.75, 3.75, 30)
    v[3, 0, 3], v[3, 0, 40] = math.inf, -math.inf
    v[4, 0, 5], v[4, 0, 6] = math.nan, 1e30
    v[5] *= 1e-7                                   # scales below fp16's normal range
    lib.append(c.cache, c.batch, None, v.cuda(), v.cuda())
    lib.moe.sync()
    k, w = lib.read(c.cache, c.batch, 6, torch.float32)
    assert torch.equal(k, w) and torch.isfinite(k).all()
    x = v.nan_to_num(0.0, 65504.0, -65504.0).clamp(-65504, 65504).view(6, 2, 32)
    hi, lo = x.amax(-1), x.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) * -0.125).half().float()[..., None]
    inv = torch.where(d != 0, 1 / d, 0.0)
    want = ((x * inv + 8.5).floor().clamp(0, 15) - 8) * d
    assert torch.equal(k.cpu().view(6, 2, 32), want)
    assert k[2, 0, 0] == 4.0 and k[2, 0, 1] == -3.5 and k[3, 0, 3] == 65504 and k[3, 0, 40] == -65504


def test_append_parts_in_place_and_alone(lib):
    from laii_b200.attn import Rope
    c = Case([(3, 10)], 16, 2, 64, fill=False)
    g = gen(3)
    ang = torch.rand(10, 32, generator=g)
    rope = Rope(ang.cos().cuda(), ang.sin().cuda())
    q, k, v = (torch.randn(3, h, 64, generator=g).bfloat16().cuda() for h in (4, 2, 2))
    both = lib.append(c.cache, c.batch, q, k, v, rope)
    one = c.cache.pages.clone()
    c.cache.pages.fill_(255)
    assert lib.append(c.cache, c.batch, None, k, v, rope) is None
    assert torch.equal(c.cache.pages, one)
    c.cache.pages.fill_(255)
    assert torch.equal(lib.append(c.cache, c.batch, q, None, None, rope), both)
    assert (c.cache.pages == 255).all()
    lib.append(c.cache, c.batch, q, k, v, rope, q_out=q)
    assert torch.equal(q, both)
    plain = lib.append(c.cache, c.batch, q, k, v)   # no rotation at all
    assert torch.equal(plain, q)
    lib.moe.sync()


@pytest.mark.parametrize("what", ["page", "table", "rope"])
def test_append_out_of_range_is_reported(lib, what):
    from laii_b200.attn import Rope
    from laii_b200.moe import MoEError
    c = Case([(2, 20), (1, 5)], 16, 1, 64, fill=False)
    rope = None
    if what == "page":
        c.batch._keep[2][0, 1] = 999
    elif what == "table":
        c.batch._keep[1][0] = 500
    else:
        rope = Rope(torch.ones(19, 32, device="cuda"), torch.zeros(19, 32, device="cuda"))
    k = torch.randn(3, 1, 64, generator=gen(1)).cuda()
    lib.append(c.cache, c.batch, None, k, k, rope)
    with pytest.raises(MoEError) as e:
        lib.moe.sync()
    assert e.value.status == -10
    c.rows = [(0, 0), (1, 5)]
    got = ref.split_page(c.cache.pages.cpu(), 16, 1, 64)
    page = int(c.table[1, 0])
    want, _ = ref.quantise(k[2].cpu())
    assert torch.allclose(ref.unpack_head(got[0][page, :, 4], got[1][page, :, 4]), want, atol=1e-6)
    lib.moe.sync()


# ---- together -------------------------------------------------------------------------------------------------------


def test_append_then_attend_token_by_token_equals_the_prompt(lib):
    """A prompt at once and the same tokens one by one leave the same cache and, within rounding, the same rows."""
    from laii_b200.attn import KVBatch, KVPages, Rope
    n, H, hkv, D, P = 70, 8, 2, 64, 16
    g = gen(12)
    ang = torch.rand(n, 32, generator=g) * 6
    rope = Rope(ang.cos().cuda(), ang.sin().cuda(), q_norm=torch.ones(64).cuda(), k_norm=torch.ones(64).cuda())
    q, k, v = (torch.randn(n, h, D, generator=g).bfloat16().cuda() for h in (H, hkv, hkv))
    table = torch.arange(5, dtype=torch.int32, device="cuda").flip(0).view(1, 5).contiguous()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    whole, step = KVPages.empty(5, P, hkv, D), KVPages.empty(5, P, hkv, D)
    whole.pages.zero_(), step.pages.zero_()
    bt = KVBatch(i32(0, n), i32(n), table)
    a = lib.attend(whole, bt, lib.append(whole, bt, q, k, v, rope))
    rows = []
    for i in range(n):
        bi = KVBatch(i32(0, 1), i32(i + 1), table)
        rows.append(lib.attend(step, bi, lib.append(step, bi, q[i:i + 1], k[i:i + 1], v[i:i + 1], rope)))
    lib.moe.sync()
    assert torch.equal(whole.pages, step.pages)
    b = torch.cat(rows)
    assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * a.float().abs() + 2.0 ** -8).all()
