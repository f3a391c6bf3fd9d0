"""Attention over the 4-bit cache where a call has enough rows for the tensor-core kernel: heads and tokens that make
hundreds of 32-row units, against the same plain formulas in 64 bits and under the same bounds as the smaller calls."""
import pytest
import torch

from test_attn_ops import DTYPES, Case, check_attend, gen, lib  # noqa: F401

pytestmark = pytest.mark.gpu

RAGGED = [(130, 130), (1, 1), (67, 200), (300, 300)]
SPLIT = [(200, 2100)]                          # few tiles of long walks: their keys in parts
SPLIT_RAGGED = [(100, 3000), (0, 40), (90, 95), (1, 2000), (70, 1500)]  # parts that short walks do not have


def run(lib, rows, P, hkv, G, D, name="bf16", seed=0, mul=0.7, **kw):  # noqa: F811
    c = Case(rows, P, hkv, D, seed=seed)
    q = (torch.randn(c.T, hkv * G, D, generator=gen(seed + 7)) * mul).to(DTYPES[name])
    out = lib.attend(c.cache, c.batch, q.cuda(), **kw)
    lib.moe.sync()
    check_attend(c, q, out, name, kw.pop("scale", D ** -0.5), **kw)
    return c, q, out


@pytest.mark.parametrize("rows", [RAGGED, SPLIT, SPLIT_RAGGED], ids=["ragged", "split", "split_ragged"])
@pytest.mark.parametrize("P,hkv,G,D,name", [(16, 16, 4, 64, "bf16"), (64, 8, 4, 64, "f32"), (128, 8, 5, 128, "f16"),
                                            (32, 8, 8, 128, "bf16"), (64, 4, 16, 64, "f16")])
def test_types_pages_and_groups(lib, rows, P, hkv, G, D, name):  # noqa: F811
    c, q, out = run(lib, rows, P, hkv, G, D, name, seed=D + P)
    assert torch.equal(out, lib.attend(c.cache, c.batch, q.cuda()))  # the same bits again


@pytest.mark.parametrize("rows", [RAGGED, SPLIT_RAGGED], ids=["ragged", "split"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=1), dict(window=33), dict(window=100000), dict(softcap=2.0),
                                dict(softcap=30.0, window=1100), dict(causal=False, softcap=5.0)])
def test_masks_and_caps(lib, rows, D, kw):  # noqa: F811
    run(lib, rows, 32, 8, 6, D, seed=D, scale=0.11, **kw)


@pytest.mark.parametrize("rows", [[(300, 900)], [(128, 2500)]])
@pytest.mark.parametrize("scale", [4.0, -4.0, 1e-4, 0.0])
def test_growing_scores(lib, rows, scale):  # noqa: F811
    """The running maximum moves many times, by much; parts whose maxima are far apart."""
    run(lib, rows, 16, 16, 4, 64, seed=11, mul=1.0, scale=scale)


def test_rows_that_see_no_key(lib):  # noqa: F811
    """More rows than tokens: the first see nothing and are zero."""
    rows = [(400, 130), (200, 0), (300, 2000)]
    c = Case(rows, 64, 8, 64, seed=2)
    q = torch.randn(c.T, 32, 64, generator=gen(5)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda())
    lib.moe.sync()
    check_attend(c, q, out, "bf16", 0.125)
    assert (out[:270] == 0).all() and (out[400:600] == 0).all()


def test_strides_another_stream_and_any_hint(lib):  # noqa: F811
    c = Case([(400, 1200), (70, 70)], 64, 8, 64, seed=1)
    fused = torch.randn(c.T + 3, 36, 64, generator=gen(3)).bfloat16().cuda()
    q = fused[:, 2:34]
    out = torch.full((c.T + 3, 34, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lib.attend(c.cache, c.batch, q, out=out[:, 1:33])
    s.synchronize()
    lib.moe.sync()
    check_attend(c, q, out[:, 1:33], "bf16", 0.125)
    assert (out[c.T:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 33] == 7).all()
    for hint in (1, 0, 10 ** 6):
        c.batch._c.max_kv_len = hint
        check_attend(c, q, lib.attend(c.cache, c.batch, q), "bf16", 0.125)


def test_two_streams_share_the_parts(lib):  # noqa: F811
    c = Case(SPLIT, 64, 8, 64, seed=6)
    qs = [torch.randn(c.T, 32, 64, generator=gen(8 + i)).bfloat16().cuda() for i in range(2)]
    want = [lib.attend(c.cache, c.batch, q) for q in qs]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(lib.attend(c.cache, c.batch, qs[i % 2]))
    torch.cuda.synchronize()
    lib.moe.sync()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))


def test_a_graph_follows_the_lengths(lib):  # noqa: F811
    c = Case(SPLIT, 64, 8, 64, seed=2)
    q = torch.randn(c.T, 32, 64, generator=gen(1)).bfloat16().cuda()
    out = torch.empty_like(q)
    lib.reserve()
    lib.attend(c.cache, c.batch, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lib.attend(c.cache, c.batch, q, out=out)
    for n in (2100, 500, 1533, 200):
        c.rows[0] = (200, n)
        c.batch._keep[1].fill_(n)
        g.replay()
        torch.cuda.synchronize()
        check_attend(c, q, out, "bf16", 0.125)
    lib.moe.sync()


@pytest.mark.parametrize("what", ["page", "table", "offsets", "length"])
def test_a_batch_out_of_range_is_reported(lib, what):  # noqa: F811
    """Nothing outside the rows is touched, the sequence before the bad one is right, and the next call works."""
    from laii_b200.moe import MoEError
    c = Case([(400, 400), (300, 900)], 16, 8, 64, seed=4)
    if what == "page":
        t = c.table.clone()
        t[1, 3] = 10 ** 6
        c.batch._keep[2].copy_(t)
    elif what == "table":
        c.batch._keep[1].copy_(torch.tensor([400, 2000], dtype=torch.int32))
    elif what == "length":
        c.batch._keep[1].copy_(torch.tensor([400, -7], dtype=torch.int32))
    else:
        c.batch._keep[0].copy_(torch.tensor([0, 400, 2 ** 31 - 1], dtype=torch.int32))
    q = torch.randn(c.T, 32, 64, generator=gen(6)).bfloat16()
    buf = torch.full((c.T + 2, 32, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    lib.attend(c.cache, c.batch, q.cuda(), out=buf[1:-1])
    with pytest.raises(MoEError) as e:
        lib.moe.sync()
    assert e.value.status == -10
    assert (buf[0] == 5).all() and (buf[-1] == 5).all()
    c.rows = c.rows[:1]
    check_attend(c, q, buf[1:-1], "bf16", 0.125)
    lib.moe.sync()
    run(lib, [(400, 400)], 16, 8, 4, 64)


@pytest.mark.parametrize("n,q", [(300, 1), (700, 2)])
def test_more_sequences_than_threads(lib, n, q):  # noqa: F811
    """Batches that a block looks through in several passes; some sequences without rows or without tokens."""
    rows = [(0 if b % 11 == 5 else q, 0 if b % 7 == 3 else 1 + (b * 37) % 90) for b in range(n)]
    run(lib, rows, 16, 2, 4, 64, seed=3)
    run(lib, rows + [(330, 900)] + rows[:40], 16, 8, 4, 64, seed=4)


def test_a_closed_handle_is_refused():
    from laii_b200.attn import GpuAttn
    from laii_b200.moe import GpuMoE
    moe = GpuMoE(0)
    attn = GpuAttn(moe)
    moe.close()
    with pytest.raises(ValueError):
        attn.add_rmsnorm(torch.zeros(2, 256, device="cuda"), None, None)
    with pytest.raises(ValueError):
        attn.reserve()
