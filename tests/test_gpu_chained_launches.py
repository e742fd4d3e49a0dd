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
