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
