"""Attention-side calls after errors, on broken batches, freed pages and odd values: what they report, and that the rest
stays right."""
import pytest
import torch

from test_attn_ops import Case, check_attend, gen, lib  # noqa: F401

pytestmark = pytest.mark.gpu


def device_check(lib):  # noqa: F811
    """The next sync reports what a kernel found out of range, once."""
    from laii_b200.moe import MoEError
    with pytest.raises(MoEError) as e:
        lib.moe.sync()
    assert e.value.status == -10
    lib.moe.sync()


def bad_page(c):
    t = c.table.clone()
    t[0, 1] = 10 ** 6
    c.batch._keep[2].copy_(t)


# ---- calls after an error: the counters of split work are cleared while nothing uses them ------------------------


@pytest.mark.parametrize("rows,hkv", [([(1, 20000)], 1), ([(200, 2100)], 8)], ids=["rows", "tiles"])
def test_split_calls_right_after_a_reported_error(lib, rows, hkv):  # noqa: F811
    c, bad = Case(rows, 64, hkv, 64, seed=6), Case([(1, 300)], 64, 1, 64, seed=7)
    bad_page(bad)
    q = torch.randn(c.T, 4 * hkv, 64, generator=gen(8)).bfloat16().cuda()
    qb = torch.randn(1, 4, 64, generator=gen(9)).bfloat16().cuda()
    want = lib.attend(c.cache, c.batch, q)
    check_attend(c, q, want, "bf16", 0.125)
    side, outs = torch.cuda.Stream(), []
    for _ in range(20):
        lib.attend(bad.cache, bad.batch, qb)
        device_check(lib)
        with torch.cuda.stream(side):
            outs += [lib.attend(c.cache, c.batch, q) for _ in range(3)]
        side.synchronize()
    lib.moe.sync()
    assert all(torch.equal(o, want) for o in outs)


def test_an_error_read_by_a_forward_while_split_calls_run(lib):  # noqa: F811
    """A forward of host rows waits for its own stream only and reports the handle's error: calls that run on another
    stream meanwhile keep their counters."""
    from laii_b200 import synth
    from laii_b200.moe import MoEError
    L = synth.make_moe_layer(512, 8, 2, 512, layer=0)
    x = synth.make_hidden(3, 512, seed_offset=3)
    lib.moe.upload_layer(0, L)
    c, bad = Case([(1, 20000)], 64, 1, 64, seed=6), Case([(1, 300)], 64, 1, 64, seed=7)
    bad_page(bad)
    q = torch.randn(1, 4, 64, generator=gen(8)).bfloat16().cuda()
    want = lib.attend(c.cache, c.batch, q)
    torch.cuda.synchronize()
    side, outs = torch.cuda.Stream(), []
    for _ in range(10):
        lib.attend(bad.cache, bad.batch, q)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            outs += [lib.attend(c.cache, c.batch, q) for _ in range(30)]
        with pytest.raises(MoEError) as e:
            lib.moe.forward(0, x)
        assert e.value.status == -10
        side.synchronize()
    lib.moe.sync()
    assert all(torch.equal(o, want) for o in outs)


# ---- offsets that describe no batch --------------------------------------------------------------------------------


@pytest.mark.parametrize("hkv,G,rows", [(1, 4, (1, 50)), (8, 4, (400, 400)), (8, 4, (200, 2100))], ids=["rows", "tiles", "split"])
@pytest.mark.parametrize("start", [[0, 2 ** 31 - 1], [-1, 1], [1, 0], [0, 401]])
def test_attend_reports_the_offsets_of_one_sequence(lib, hkv, G, rows, start):  # noqa: F811
    c = Case([rows], 64, hkv, 64, seed=4)
    c.batch._keep[0].copy_(torch.tensor(start, dtype=torch.int32))
    buf = torch.full((c.T + 2, hkv * G, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    lib.attend(c.cache, c.batch, torch.randn(c.T, hkv * G, 64, generator=gen(1)).bfloat16().cuda(), out=buf[1:-1])
    device_check(lib)
    assert (buf == 5).all()


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("bad", [1, -1])
def test_attend_reports_one_bad_sequence_of_several(lib, n, bad):  # noqa: F811
    """Wherever it stands; the sequences before it are right."""
    rows = [(90, 400)] * n
    at = n - 1 if bad < 0 else 1
    c = Case(rows, 64, 8, 64, seed=4)
    c.batch._keep[0][at + 1:] = c.T + 1
    q = torch.randn(c.T, 32, 64, generator=gen(1)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda())
    device_check(lib)
    c.rows = rows[:at]
    check_attend(c, q, out, "bf16", 0.125)


@pytest.mark.parametrize("n,start", [(4, [0, 10]), (4, [-2, 4]), (4, [3, 1]), (300, [0, 2 ** 31 - 1]), (600, [0, 601])])
def test_append_and_read_report_offsets_and_leave_the_rows(lib, n, start):  # noqa: F811
    """No token of an older place is written over, and nothing is read in its name."""
    c = Case([(n, n + 40)], 16, 8, 64, fill=False)
    c.batch._keep[0].copy_(torch.tensor(start, dtype=torch.int32))
    k = torch.randn(n, 8, 64, generator=gen(1)).bfloat16().cuda()
    q = torch.randn(n, 16, 64, generator=gen(2)).bfloat16().cuda()
    before, out = c.cache.pages.clone(), torch.full_like(q, 3.0)
    lib.append(c.cache, c.batch, q, k, k, q_out=out)
    device_check(lib)
    assert torch.equal(c.cache.pages, before) and (out == 3).all()
    lib.read(c.cache, c.batch, n, torch.float32)
    device_check(lib)


@pytest.mark.parametrize("n", [3, 70, 600])
def test_append_and_read_report_one_bad_sequence_of_several(lib, n):  # noqa: F811
    c = Case([(1, 9)] * n, 16, 2, 64, fill=False)
    c.batch._keep[0][n] = n + 1  # the last sequence: two rows of a call that has one for it
    k = torch.randn(n, 2, 64, generator=gen(1)).bfloat16().cuda()
    lib.append(c.cache, c.batch, None, k, k)
    device_check(lib)
    got, _ = lib.read(c.cache, c.batch, n, torch.float32)
    device_check(lib)
    from attn_ref import quantise
    want = torch.stack([quantise(x)[0] for x in k[:n - 1].cpu().double()])
    # without a norm or a rotation the codes are exact but for the fp32 quotient at a boundary
    assert ((got[:n - 1].cpu().double() - want).abs() <= 1e-6).float().mean() > 0.999
    last = int(c.table[n - 1, 0])
    assert (c.cache.pages[last] == 255).all()


def test_padding_rows_are_no_error(lib):  # noqa: F811
    """Rows outside every sequence are padding: left alone, and nothing is reported."""
    c = Case([(2, 20), (0, 5), (3, 30)], 16, 2, 64)
    k = torch.randn(c.T + 6, 2, 64, generator=gen(1)).bfloat16().cuda()
    q = torch.randn(c.T + 6, 4, 64, generator=gen(2)).bfloat16().cuda()
    out = torch.full_like(q, 3.0)
    lib.append(c.cache, c.batch, q, k, k, q_out=out)
    lib.read(c.cache, c.batch, c.T + 6, torch.float32)
    lib.attend(c.cache, c.batch, q)
    lib.moe.sync()
    assert torch.equal(out[:c.T], q[:c.T]) and (out[c.T:] == 3).all()


# ---- lengths that the page table has no room for -------------------------------------------------------------------


@pytest.mark.parametrize("rows", [[(1, 100)], [(300, 400)], [(60, 2000), (300, 400)], [(1, 70), (1, 100)]],
                         ids=["one", "tiles", "both", "batch"])
@pytest.mark.parametrize("over", [1, 500, 2 ** 31 - 1])
def test_attend_passes_over_a_length_beyond_the_table(lib, rows, over):  # noqa: F811
    """The last sequence's length is past the table's span: reported, its rows left alone, the others right."""
    c = Case(rows, 16, 8, 64, seed=4)
    span = c.table.shape[1] * 16
    c.batch._keep[1][-1] = min(span + over, 2 ** 31 - 1)
    q = torch.randn(c.T, 32, 64, generator=gen(6)).bfloat16()
    out = torch.full((c.T, 32, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    lib.attend(c.cache, c.batch, q.cuda(), out=out)
    device_check(lib)
    assert (out[c.starts[-2]:] == 5).all()
    c.rows = rows[:-1]
    check_attend(c, q, out, "bf16", 0.125)


@pytest.mark.parametrize("rows", [[(1, 100), (0, 40)], [(300, 400), (0, 40)]])
@pytest.mark.parametrize("n", [10 ** 6, -3])
def test_the_length_of_a_sequence_without_rows_does_not_matter(lib, rows, n):  # noqa: F811
    c = Case(rows, 16, 8, 64, seed=4)
    c.batch._keep[1][1] = n
    q = torch.randn(c.T, 32, 64, generator=gen(6)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda())
    lib.moe.sync()
    c.rows = rows[:1]
    check_attend(c, q, out, "bf16", 0.125)


def test_a_length_that_fills_the_table_is_right(lib):  # noqa: F811
    c = Case([(2, 128), (130, 256)], 16, 8, 64, seed=4)
    assert c.table.shape[1] * 16 == 256
    q = torch.randn(c.T, 32, 64, generator=gen(6)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda())
    lib.moe.sync()
    check_attend(c, q, out, "bf16", 0.125)


# ---- pages behind a sliding window ----------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,hkv", [([(1, 333), (3, 261), (1, 129), (1, 17)], 2), ([(1, 5000), (1, 700)], 1), ([(8, 2000), (8, 900)], 2),
                                      ([(300, 900), (70, 611)], 8), ([(200, 2100)], 8)], ids=["decode", "long", "verify", "tiles", "split"])
@pytest.mark.parametrize("D,P", [(64, 16), (64, 32), (128, 16), (128, 64)])
@pytest.mark.parametrize("window", [1, 33, 1100])
@pytest.mark.parametrize("what", ["gone", "anything"])
def test_pages_behind_the_window_may_be_given_back(lib, rows, hkv, D, P, window, what):  # noqa: F811
    """Entries of pages that end before the first token that a row sees: -1, or a page of NaN scales."""
    c = Case(rows, P, hkv, D, seed=D + P, spare=1)
    t = c.table.clone()
    used = set(int(i) for i in t[t >= 0])
    spare = next(i for i in range(c.pages.shape[0]) if i not in used)   # all bytes 0xFF
    for b, (q, n) in enumerate(rows):
        t[b, : max(0, n - q + 1 - window) // P] = -1 if what == "gone" else spare
    c.batch._keep[2].copy_(t)
    q = torch.randn(c.T, 4 * hkv, D, generator=gen(9)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda(), window=window)
    lib.moe.sync()
    check_attend(c, q, out, "bf16", D ** -0.5, window=window)


# ---- caps far above and below the scores ----------------------------------------------------------------------------


@pytest.mark.parametrize("rows,hkv", [([(1, 300), (3, 150)], 2), ([(8, 700)], 2), ([(130, 400)], 8), ([(200, 2100)], 8)],
                         ids=["decode", "verify", "tiles", "split"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [1e-39, 0.5, 100.0, 127.9, 300.0, 1e4, 1e6, 1e9, 1e30])
def test_any_cap(lib, rows, hkv, D, cap):  # noqa: F811
    """Under the bound of scores without a cap: a large one adds an error relative to a score, not to itself."""
    import attn_ref as ref
    c = Case(rows, 32, hkv, D, seed=D)
    q = torch.randn(c.T, 4 * hkv, D, generator=gen(9)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda(), scale=0.3, softcap=cap)
    lib.moe.sync()
    assert torch.isfinite(out).all()
    for b, (n, _) in enumerate(rows):
        a = slice(c.starts[b], c.starts[b] + n)
        K, V = c.kv(b)
        want, _ = ref.attend(q[a], K, V, 0.3, softcap=cap)
        _, tol = ref.attend(q[a], K, V, 0.3)
        # the bound's weights are those of uncapped scores: the capped ones are flatter, so by the largest value instead.
        # A score is off by 2^-11 |q| |k| scale (q and the keys rounded; tanh's slope is at most one) and, up to a cap of
        # 128, by 2^-22 of that; a probability by twice that, 2^-11 of itself and 2^-25 where fp16 goes subnormal
        dz = torch.einsum("nhgd,jhd->nhgj", q[a].double().view(n, hkv, 4, D).abs(), K.abs()).amax(-1) * 0.3 * (2.0 ** -11 + 2.0 ** -19) + 128 * 2.0 ** -22
        t = ((2.0 ** -10 + 2 * dz + 2.0 ** -17 + len(K) * 2.0 ** -25) * V.abs().amax()).reshape(n, -1, 1)
        if cap >= 1e6:  # |z| / cap so small that the weights are those of the bound
            t = torch.minimum(t, tol * 1.01 + 1e-9)
        err = (out[a].cpu().double() - want).abs()
        assert (err <= t + 2.0 ** -8 * want.abs()).all(), float((err / (t + 2.0 ** -8 * want.abs())).max())


@pytest.mark.parametrize("rows,hkv", [([(1, 300)], 2), ([(130, 400)], 8)], ids=["rows", "tiles"])
def test_a_cap_beyond_all_scores_is_none(lib, rows, hkv):  # noqa: F811
    c = Case(rows, 32, hkv, 64, seed=1)
    q = torch.randn(c.T, 4 * hkv, 64, generator=gen(9)).bfloat16().cuda()
    plain = lib.attend(c.cache, c.batch, q)
    assert torch.equal(lib.attend(c.cache, c.batch, q, softcap=1e37), plain)
    lib.moe.sync()


# ---- one key far above all others -----------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,hkv,G", [((1, 6000), 1, 4), ((8, 6000), 1, 4), ((64, 20000), 8, 4), ((1200, 6000), 8, 4)],
                         ids=["decode", "verify", "split", "tiles"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nats", [10.0, 17.5, 20.0])
def test_keys_far_below_one_keep_their_part(lib, rows, hkv, G, D, nats):  # noqa: F811
    """The first key scores `nats` and has a value of 0, all others score 0 and have 1: row i sees n = i of them and is
    n e^-nats / (1 + n e^-nats).  q, keys and values are exact.  A probability is off by 2^-11 of itself (fp16) and 2^-20
    (its exponent, 25 at most, in fp32), or by 2^-32 of the largest where fp16 goes subnormal, 2^-25 of a reference 2^7
    below the largest score."""
    n, length = rows
    c = Case([(length, length)], 64, hkv, D, fill=False)
    k = torch.zeros(length, hkv, D)
    v = torch.ones(length, hkv, D)
    k[0], v[0] = 1.0, 0.0
    lib.append(c.cache, c.batch, None, k.cuda(), v.cuda())
    c.batch._keep[0][1] = n
    q = torch.ones(n, hkv * G, D, device="cuda")
    scale = nats / D
    out = lib.attend(c.cache, c.batch, q, scale=scale).cpu().double()
    lib.moe.sync()
    seen = torch.arange(length - n, length, dtype=torch.float64)[:, None, None]
    part = seen * torch.exp(torch.tensor(-nats, dtype=torch.float64))
    want = part / (1 + part)
    assert ((out - want).abs() <= want * (2.0 ** -10 + 2.0 ** -19) + seen * 2.0 ** -32).all(), float(((out - want).abs() / want).max())


@pytest.mark.parametrize("rows,hkv", [([(1, 900)], 2), ([(8, 900)], 2), ([(300, 900)], 8), ([(200, 2100)], 8)],
                         ids=["decode", "verify", "tiles", "split"])
@pytest.mark.parametrize("scale", [0.02, 0.6, -3.0, 40.0])
def test_scores_that_climb(lib, rows, hkv, scale):  # noqa: F811
    """Keys in the order of their scores, so that the reference moves late and often: no probability leaves fp16."""
    c = Case(rows, 16, hkv, 64, seed=5)
    import attn_ref as ref
    kc, ks, _, _ = ref.split_page(c.pages, 16, hkv, 64)
    p = c.pages.view(c.pages.shape[0], hkv, -1)
    for i, page in enumerate(c.table[0]):   # scales that grow from key to key
        at = (torch.arange(16) + 16 * i + 1.0) / rows[0][1]
        p[int(page), :, 512:576] = (0.1 * at)[:, None].expand(16, 2).half().contiguous().view(torch.uint8).reshape(-1)
    c.cache.pages.copy_(c.pages)
    q = torch.randn(c.T, 4 * hkv, 64, generator=gen(3)).bfloat16()
    out = lib.attend(c.cache, c.batch, q.cuda(), scale=scale)
    lib.moe.sync()
    check_attend(c, q, out, "bf16", scale)


# ---- one handle, streams that share a name --------------------------------------------------------------------------


def test_per_thread_default_streams_take_turns(lib):  # noqa: F811
    """Two threads' default streams have one handle value (cudaStreamPerThread): a call of the second waits for the work
    that the first's has on the scratch."""
    import ctypes
    import threading
    c = Case([(1, 20000)], 64, 1, 64, seed=6)
    q = torch.randn(1, 4, 64, generator=gen(8)).bfloat16().cuda()
    want = lib.attend(c.cache, c.batch, q)
    outs = [torch.zeros_like(q) for _ in range(2)]
    done = [torch.cuda.Event() for _ in range(2)]
    c.batch.rows(1)
    torch.cuda.synchronize()

    def work(i, spin):
        s = torch.cuda.ExternalStream(2)  # cudaStreamPerThread
        with torch.cuda.stream(s):
            if spin:
                torch.cuda._sleep(200_000_000)  # some 0.1 s of clocks
            st = lib._lib.lfm_gpu_attn_forward(lib.moe._h, ctypes.byref(c.cache._c), ctypes.byref(c.batch._c), 4, 0.125, 1, 0, 0.0,
                                               30, q.data_ptr(), 256, outs[i].data_ptr(), 256, ctypes.c_void_p(2))
            done[i].record()
        status.append(st)

    status = []
    for i, spin in enumerate((True, False)):
        t = threading.Thread(target=work, args=(i, spin))
        t.start()
        t.join()
    done[1].synchronize()
    assert done[0].query()  # the first thread's work is over too
    torch.cuda.synchronize()
    lib.moe.sync()
    assert status == [0, 0] and all(torch.equal(o, want) for o in outs)


def test_a_stream_made_after_another_was_destroyed_waits(lib):  # noqa: F811
    """Whatever value the new stream's handle has."""
    import ctypes
    cudart = torch.cuda.cudart()
    c = Case([(1, 20000)], 64, 1, 64, seed=6)
    q = torch.randn(1, 4, 64, generator=gen(8)).bfloat16().cuda()
    want = lib.attend(c.cache, c.batch, q)
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        box = ctypes.c_size_t()
        err = cudart.cudaStreamCreate(ctypes.addressof(box))
        assert int(err) == 0
        s = torch.cuda.ExternalStream(box.value)
        with torch.cuda.stream(s):
            torch.cuda._sleep(2_000_000)
            outs.append(lib.attend(c.cache, c.batch, q))
        assert int(cudart.cudaStreamDestroy(box.value)) == 0   # with its work under way
    torch.cuda.synchronize()
    lib.moe.sync()
    assert all(torch.equal(o, want) for o in outs)


# ---- NaN and infinities ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("D", [256, 1024])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_add_rmsnorm_keeps_what_is_not_finite(lib, D, value):  # noqa: F811
    """A NaN spreads over its row, an infinity leaves a NaN in its place (its row's norm is infinite): the Q8_K values say
    so as the other outputs do, and the other rows are as without it."""
    x = torch.randn(5, D, generator=gen(1))
    w = 1 + 0.1 * torch.randn(D, generator=gen(2))
    _, xb0, q0 = lib.add_rmsnorm(x.cuda(), None, w.cuda(), xb_dtype=torch.float32)
    x[2, 7] = value
    xo, xb, q8 = lib.add_rmsnorm(x.cuda(), None, w.cuda(), xb_dtype=torch.float32)
    lib.moe.sync()
    assert torch.equal(xo.cpu().nan_to_num(7.0), x.nan_to_num(7.0)) and xb[2, 7].isnan()
    v = lib.read_q8(q8, torch.float32)
    blocks = xb[2].view(-1, 256).isnan().any(1)
    assert blocks[0] and torch.equal(v[2].view(-1, 256).isnan().all(1), blocks)
    assert not v[2].view(-1, 256)[~blocks].isnan().any()
    others = [0, 1, 3, 4]
    assert torch.equal(xb[others], xb0[others]) and torch.equal(q8[others], q0[others])


def test_add_rmsnorm_infinite_weight(lib):  # noqa: F811
    x = torch.randn(2, 512, generator=gen(1)).cuda()
    w = torch.ones(512)
    w[300] = float("inf")
    q8 = lib.add_rmsnorm(x, None, w.cuda())[2]
    v = lib.read_q8(q8, torch.float32)
    assert torch.isfinite(v[:, :256]).all() and not torch.isfinite(v[:, 256:]).any()
    assert torch.equal(q8[:, 0], lib.add_rmsnorm(x, None, None)[2][:, 0])


@pytest.mark.parametrize("rows,hkv", [([(1, 300), (1, 90)], 2), ([(8, 700)], 2), ([(130, 400)], 8), ([(200, 2100)], 8), ([(400, 900)], 8)],
                         ids=["decode", "verify", "tiles", "split", "more"])
@pytest.mark.parametrize("kw", [dict(), dict(softcap=20.0), dict(window=50)], ids=["plain", "cap", "window"])
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_attend_nan_and_infinite_q(lib, rows, hkv, kw, name):  # noqa: F811
    """A NaN makes its own row NaN, infinities stand for +-65504; every other row is the same, bit for bit."""
    from test_attn_ops import DTYPES
    c = Case(rows, 32, hkv, 64, seed=3)
    H = 4 * hkv
    q = torch.randn(c.T, H, 64, generator=gen(9)).to(DTYPES[name])
    big = torch.tensor(65504.0).to(DTYPES[name])
    q[c.T - 1, 1, 3], q[0, H - 2, 60] = big, -big
    want = lib.attend(c.cache, c.batch, q.cuda(), **kw)
    assert torch.isfinite(want).all()
    q[c.T - 1, 1, 3], q[0, H - 2, 60] = float("inf"), float("-inf")
    nan = (c.T // 2, 2)
    q[nan[0], nan[1], 11] = float("nan")
    out = lib.attend(c.cache, c.batch, q.cuda(), **kw)
    lib.moe.sync()
    assert out[nan].isnan().all()
    keep = torch.ones(c.T, H, dtype=torch.bool, device="cuda")
    keep[nan] = False
    assert torch.equal(out[keep], want[keep])
