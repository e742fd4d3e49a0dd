"""Launches that depend programmatically on the one before them (VW_DECODE_PDL, VW_PREFILL_PDL) see all of its work.

A decode is followed by its combine grid, and a dependent launch waits for the combine alone.  In a batch that no CTA range
cuts (every sequence in one page) the combine has nothing to merge, and must still not complete before the decode: the next
launch reads the rows that the decode appended, over slots that held NaN patterns.
"""
import pytest

torch = pytest.importorskip("torch")
from tests.paged_cases import Batch, attend, check, held  # noqa: E402

pytestmark = pytest.mark.gpu

KINDS = [("bf16", "bf16", 128, 28, 4, 0), ("bf16", "bf16", 128, 28, 4, 20), ("f16", "f16", 64, 14, 2, 7),
         ("fp8", "bf16", 128, 32, 8, 0), ("fp8", "f16", 128, 16, 2, 9), ("fp4", "bf16", 128, 32, 8, 0),
         ("fp4", "f16", 64, 16, 1, 12)]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def poison(bt):
    bt.pool.pages_u8().fill_(0xFF)
    if bt.kv == "fp8":
        bt.pool.scales_f32().fill_(float("nan"))


@pytest.mark.parametrize("kv,io,D,Hq,Hkv,window", KINDS)
def test_reads_what_an_unsplit_decode_appended(kv, io, D, Hq, Hkv, window):
    from voidweb_b200 import _lib as C
    totals = [1 + i % 16 for i in range(300)]
    bt = Batch(31, kv, io, D, Hq, Hkv, totals, layers=2, max_batch=300)
    table, lens = bt.device_table(), bt.lens()
    q, q2 = bt.rows(bt.B, Hq).to(bt.dev), bt.rows(bt.B, Hq).to(bt.dev)
    kn, vn = (torch.stack([x[-1] for x in y]).to(bt.dev) for y in (bt.k, bt.v))
    cu, start = torch.arange(bt.B + 1, dtype=torch.int32, device=bt.dev), lens - 1
    none = torch.zeros_like(lens)
    win = dict(window=window, sinks=1) if window else {}
    a, b, c = (torch.zeros_like(q) for _ in range(3))
    got = {}
    for how in ("waited", "prefill", "decode", "no pages"):
        poison(bt)
        bt.fill([n - 1 for n in totals])
        torch.cuda.synchronize()
        for x in (a, b, c):
            x.fill_(7.0)
        bt.pool.paged_decode(0, q, table, lens, a, k_new=kn, v_new=vn, **win)
        if how == "waited":
            torch.cuda.synchronize()
            bt.pool.paged_prefill(0, q2, cu, start, table, b, **win)
            bt.pool.paged_decode(0, q2, table, lens, c, **win)
            assert bt.pool.check() == 0
        elif how == "prefill":
            bt.pool.paged_prefill(0, q2, cu, start, table, b, flags=C.VW_PREFILL_PDL, **win)
            assert bt.pool.check() == 0
        elif how == "decode":
            bt.pool.paged_decode(0, q2, table, lens, c, flags=C.VW_DECODE_PDL, **win)
            assert bt.pool.check() == 0
        else:          # a batch of no pages between them, of another layer (flagged, writes nothing)
            bt.pool.paged_decode(1, q, table, none, c, flags=C.VW_DECODE_PDL | C.VW_DECODE_EARLY_PAGES, **win)
            bt.pool.paged_prefill(0, q2, cu, start, table, b, flags=C.VW_PREFILL_PDL, **win)
            assert bt.pool.check() == C.VW_DEV_ERR_SEQ_LEN
            assert (c == 7.0).all()
        got[how] = [x.clone() for x in (a, b, c)]
    assert all(torch.equal(got[h][0], got["waited"][0]) for h in got)
    assert torch.equal(got["prefill"][1], got["waited"][1]) and torch.equal(got["no pages"][1], got["waited"][1])
    assert torch.equal(got["decode"][2], got["waited"][2])
    if kv != "fp8":
        for s in range(0, bt.B, 17):
            ref = attend(q2[s:s + 1].cpu(), held(bt.k[s], kv), held(bt.v[s], kv), torch.tensor([totals[s] - 1]), window, 1 if window else 0)
            check(got["prefill"][1][s:s + 1], *ref, io, kv, f"prefill {s}")
            check(got["decode"][2][s:s + 1], *ref, io, kv, f"decode {s}")


@pytest.mark.parametrize("n", [9, 700], ids=["split", "whole"])
@pytest.mark.parametrize("kv,io,D,Hq,Hkv,window", KINDS)
def test_decodes_and_prefills_in_turn(kv, io, D, Hq, Hkv, window, n):
    """Layers of a mixed step: a decode with fused append, the prefill of another sequence's chunk (over cached rows, then over
    rows that the call appends), all dependent launches, each prefill's queries the outputs of the launch before it; the bits
    of the same calls made one after the other."""
    from voidweb_b200 import _lib as C
    L, totals = 3, [3000, 40, 7, 900]
    win = dict(window=window * 30, sinks=1) if window else {}
    a, b = (Batch(32, kv, io, D, Hq, Hkv, totals, layers=L).fill([totals[0] - n, 39, 6, 899]) for _ in range(2))
    q = a.rows(3, Hq).to(a.dev)
    kn, vn = (torch.stack([x[-1] for x in y[1:]]).to(a.dev) for y in (a.k, a.v))
    kc, vc = (y[0][-n:].to(a.dev) for y in (a.k, a.v))
    cu, start = torch.tensor([0, n], dtype=torch.int32, device=a.dev), a.lens()[:1] - n
    before = torch.tensor([0, 3], dtype=torch.int32, device=a.dev), a.lens()[:1] - n - 3     # the three tokens before the chunk
    q0, results = a.rows(n, Hq).to(a.dev), []
    for bt, chained in ((a, False), (b, True)):
        t, lens = bt.device_table(), bt.lens()
        t0, t1, l1 = t[:1].contiguous(), t[1:].contiguous(), lens[1:].contiguous()
        outs = [[torch.full_like(x, 7.0) for x in (q, q, q0, q0)] for _ in range(L)]
        pdl = C.VW_PREFILL_PDL if chained else 0
        qc = q0
        torch.cuda.synchronize()

        def done():
            if not chained:
                torch.cuda.synchronize()

        for l, (dec, mid, pre, again) in enumerate(outs):
            flags = (C.VW_DECODE_PDL | C.VW_DECODE_EARLY_PAGES) if chained and l else C.VW_DECODE_PDL if chained else 0
            bt.pool.paged_decode(l, q, t1, l1, dec, k_new=kn, v_new=vn, flags=flags, **win)
            done()
            bt.pool.paged_prefill(l, dec, *before, t0, mid, flags=pdl, **win)
            done()
            bt.pool.paged_prefill(l, qc, cu, start, t0, pre, k_new=kc, v_new=vc, flags=pdl, **win)
            done()
            bt.pool.paged_prefill(l, pre, cu, start, t0, again, flags=pdl, **win)
            done()
            qc = again
        assert bt.pool.check() == 0
        results.append([x for o in outs for x in o])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    assert torch.equal(a.pool.pages_u8(), b.pool.pages_u8())
    assert all(x.isfinite().all() for x in results[0])


@pytest.mark.parametrize("kv,io,D,Hq,Hkv,window", KINDS)
def test_host_step_of_an_unsplit_batch(kv, io, D, Hq, Hkv, window):
    """The read-back of a layer's outputs follows its combine: direct, recorded and replayed steps read finished outputs."""
    L, totals = 4, [1 + i % 16 for i in range(300)]
    a, b = (Batch(33, kv, io, D, Hq, Hkv, totals, layers=L, max_batch=300).fill([n - 1 for n in totals]) for _ in range(2))
    q = torch.stack([a.rows(a.B, Hq) for _ in range(L)]).pin_memory()
    kn, vn = (torch.stack([torch.stack([x[-1] for x in y])] * L).pin_memory() for y in (a.k, a.v))
    table, lens = a.device_table().cpu().pin_memory(), a.lens().cpu().pin_memory()
    win = dict(window=window, sinks=1) if window else {}
    want = torch.zeros_like(q)
    for l in range(L):
        o = torch.zeros_like(q[l]).to(b.dev)
        b.pool.paged_decode(l, q[l].to(b.dev), b.device_table(), b.lens(), o, k_new=kn[l].to(b.dev), v_new=vn[l].to(b.dev), **win)
        torch.cuda.synchronize()
        want[l] = o.cpu()
    out = torch.zeros_like(q).pin_memory()
    for _ in range(6):
        out.fill_(7.0)
        a.pool.decode_step_host(q, kn, vn, table, lens, out, **win)
        assert torch.equal(out, want)
    assert a.pool.check() == b.pool.check() == 0
    assert torch.equal(a.pool.pages_u8(), b.pool.pages_u8())
