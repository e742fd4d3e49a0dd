"""What a window hides on 4-bit pages may hold anything: NaN scales and NaN-like codes written into the records themselves.

(A NaN row that goes through the append is quantised to zeros, and an infinite one to finite values, so bytes are the only
way to put such rows there.)  0xFF is an E4M3 NaN as a scale.
"""
import pytest

torch = pytest.importorskip("torch")
from tests.paged_cases import Batch, attend, check, held, hidden_pages  # noqa: E402

pytestmark = pytest.mark.gpu

SHAPES = [("bf16", 128, 28, 4), ("f16", 64, 14, 2), ("f16", 128, 16, 1), ("bf16", 64, 6, 6)]
WINDOWS = [(1, 0), (1, 1), (16, 0), (17, 3), (100, 4), (33, 16), (64, 40), (5, 1000), (250, 17)]
LENS = [1, 2, 15, 16, 17, 33, 100, 257, 600, 1000]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def spoil(bt, b, first, last):
    """Every byte of the records that belongs to tokens [first, last) of sequence b becomes 0xFF; returns how many tokens."""
    D, half = bt.D, 9 * bt.D
    rec = bt.pool.pages_u8().view(bt.layers, bt.nb, bt.Hkv, 18 * D)
    for p in range(first, last):
        r, t = rec[:, bt.table[b, p // 16].item()], p % 16
        for at in (0, half):
            r[:, :, at + t * (D // 2):at + (t + 1) * (D // 2)] = 0xFF
        r[:, :, 8 * D + t * (D // 16):8 * D + (t + 1) * (D // 16)] = 0xFF          # K scales: a token's groups together
        r[:, :, half + 8 * D + t:half + 9 * D:16] = 0xFF                          # V scales: a group's tokens together
    return max(0, last - first)


def test_spoiled_rows_are_no_rows():
    """The bytes reach the rows they are meant for, and no others.  (The gather's f16 -> bf16 step is for values that an append
    leaves, at most 6 * 448; it makes a NaN a larger number, where the attention's f16 keeps it.)"""
    for io, D in (("bf16", 128), ("f16", 64)):
        bt = Batch(1, "fp4", io, D, 2, 2, [40]).fill()
        spoil(bt, 0, 5, 19)
        for x, rows in zip(bt.pool.gather(0, bt.device_table()[0], 40)[:2], (bt.k[0], bt.v[0])):
            x = x.transpose(0, 1).cpu()
            assert not (x[5:19].abs() <= 2688).any() and (io == "bf16" or x[5:19].isnan().all())
            assert torch.equal(x[:5].double(), held(rows, "fp4")[:5]) and torch.equal(x[19:].double(), held(rows, "fp4")[19:])


@pytest.mark.parametrize("append", [False, True], ids=["decode", "append"])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("io,D,Hq,Hkv", SHAPES)
def test_decode(io, D, Hq, Hkv, window, sinks, append):
    bt = Batch(window + D, "fp4", io, D, Hq, Hkv, LENS).fill([n - 1 for n in LENS] if append else None)
    spoiled = sum(spoil(bt, b, min(sinks, n), max(min(sinks, n), n - window)) for b, n in enumerate(LENS))
    assert spoiled or sinks >= 1000
    table = bt.device_table(lambda b, pg: hidden_pages(LENS[b] - 1, LENS[b] - 1, window, sinks)(pg))
    q = bt.rows(bt.B, Hq)
    out = torch.full_like(q, 7.0).to(bt.dev)
    kn, vn = (torch.stack([x[-1] for x in y]).to(bt.dev) if append else None for y in (bt.k, bt.v))
    bt.pool.paged_decode(0, q.to(bt.dev), table, bt.lens(), out, k_new=kn, v_new=vn, window=window, sinks=sinks)
    assert bt.pool.check() == 0
    for b, n in enumerate(LENS):
        ref = attend(q[b:b + 1], held(bt.k[b], "fp4"), held(bt.v[b], "fp4"), torch.tensor([n - 1]), window, sinks)
        check(out[b:b + 1], *ref, io, "fp4", f"sequence {b}")


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("chunks", [[(0, 5), (16, 16), (700, 130), (31, 1)], [(3000, 9)]], ids=["4", "split"])
@pytest.mark.parametrize("io,D,Hq,Hkv", SHAPES)
def test_prefill(io, D, Hq, Hkv, chunks, window, sinks):
    """Rows that no token of the chunk sees (a tile of 128 rows may hide more of them)."""
    totals = [a + n for a, n in chunks]
    bt = Batch(len(chunks) + D, "fp4", io, D, Hq, Hkv, totals).fill([a for a, _ in chunks])
    for b, (a, n) in enumerate(chunks):
        spoil(bt, b, min(sinks, a), max(min(sinks, a), a + 1 - window))
    table = bt.device_table(lambda b, pg: hidden_pages(chunks[b][0], totals[b] - 1, window, sinks)(pg))
    q = [bt.rows(n, Hq) for _, n in chunks]
    cu = torch.tensor([0] + [n for _, n in chunks]).cumsum(0).int().to(bt.dev)
    start = torch.tensor([a for a, _ in chunks], dtype=torch.int32, device=bt.dev)
    kn = torch.cat([x[a:] for x, (a, _) in zip(bt.k, chunks)]).to(bt.dev)
    vn = torch.cat([x[a:] for x, (a, _) in zip(bt.v, chunks)]).to(bt.dev)
    qd = torch.cat(q).to(bt.dev)
    out = torch.full_like(qd, 7.0)
    bt.pool.paged_prefill(0, qd, cu, start, table, out, k_new=kn, v_new=vn, window=window, sinks=sinks)
    assert bt.pool.check() == 0
    for b, (a, n) in enumerate(chunks):
        ref = attend(q[b], held(bt.k[b], "fp4"), held(bt.v[b], "fp4"), torch.arange(a, a + n), window, sinks)
        check(out[int(cu[b]):int(cu[b + 1])], *ref, io, "fp4", f"chunk {b}")
