"""4-bit and windowed calls on streams of their own: `stream=`, and a prefill beside a decode of the same pool."""
import pytest

torch = pytest.importorskip("torch")
from tests.paged_cases import Batch, attend, check, held  # noqa: E402

pytestmark = pytest.mark.gpu

KINDS = [("fp4", "bf16", 128, 32, 8, 0), ("fp4", "f16", 64, 16, 1, 300), ("bf16", "bf16", 128, 28, 4, 2000),
         ("f16", "f16", 64, 6, 2, 5000)]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("kv,io,D,Hq,Hkv,window", KINDS)
def test_prefill_beside_decode(kv, io, D, Hq, Hkv, window):
    """A prefill that splits its tiles and a decode that splits its pages, of one pool, at the same time on two streams: the
    bits of the calls made one after the other."""
    n = 9
    totals = [6000, 7001, 500, 2333]
    bt = Batch(3, kv, io, D, Hq, Hkv, totals).fill()
    table, lens = bt.device_table(), bt.lens()
    qp, qd = bt.rows(n, Hq).to(bt.dev), bt.rows(3, Hq).to(bt.dev)
    cu = torch.tensor([0, n], dtype=torch.int32, device=bt.dev)
    start, t0, t1, l1 = lens[:1] - n, table[:1].contiguous(), table[1:].contiguous(), lens[1:].contiguous()
    win = dict(window=window, sinks=2) if window else {}
    want_p, want_d = torch.zeros_like(qp), torch.zeros_like(qd)
    bt.pool.paged_prefill(0, qp, cu, start, t0, want_p, **win)
    torch.cuda.synchronize()
    bt.pool.paged_decode(0, qd, t1, l1, want_d, **win)
    assert bt.pool.check() == 0
    outs = [(torch.zeros_like(qp), torch.zeros_like(qd)) for _ in range(40)]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for p, d in outs:
        bt.pool.paged_prefill(0, qp, cu, start, t0, p, stream=a, **win)
        bt.pool.paged_decode(0, qd, t1, l1, d, stream=b, **win)
    torch.cuda.synchronize()
    assert bt.pool.check() == 0
    assert all(torch.equal(p, want_p) and torch.equal(d, want_d) for p, d in outs)
    ref = attend(qp.cpu(), held(bt.k[0], kv), held(bt.v[0], kv), torch.arange(totals[0] - n, totals[0]), window, 2 if window else 0)
    check(want_p, *ref, io, kv, "prefill")


@pytest.mark.parametrize("kv,io,D,Hq,Hkv,window", KINDS)
def test_every_call_takes_a_stream(kv, io, D, Hq, Hkv, window):
    """All of a sequence's life on one side stream, with inputs that the stream itself produces after a long copy (a call
    on another stream would read zeros); the current stream takes no part."""
    totals = [400, 77]
    bt = Batch(4, kv, io, D, Hq, Hkv, totals)
    ref_bt = Batch(4, kv, io, D, Hq, Hkv, totals).fill()
    win = dict(window=window, sinks=2) if window else {}
    table, lens = bt.device_table(), bt.lens()
    k, v = torch.cat(bt.k).to(bt.dev), torch.cat(bt.v).to(bt.dev)
    slots = torch.cat([bt.slots(b) for b in range(2)]).to(bt.dev)
    q = bt.rows(2, Hq).to(bt.dev)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=bt.dev)
    spare = sorted(set(range(bt.nb)) - set(bt.table.flatten().tolist()))[0]
    pairs = torch.tensor([[bt.table[0, 0].item(), spare]], dtype=torch.int32, device=bt.dev)
    moved = table.clone()
    moved[0, 0] = spare
    want = torch.zeros_like(q)
    ref_bt.pool.paged_decode(0, q, table, lens, want, **win)
    big = torch.empty(1 << 28, dtype=torch.uint8, device=bt.dev)
    kk, vv, qq = torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(q)
    dec, pre = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big.fill_(1)
        for x, y in ((kk, k), (vv, v), (qq, q)):
            x.copy_(y)
    bt.pool.append(0, kk, vv, slots, stream=s)
    bt.pool.block_copy(pairs, stream=s)
    bt.pool.paged_decode(0, qq, moved, lens, dec, stream=s, **win)
    bt.pool.paged_prefill(0, qq, cu, lens - 1, moved, pre, stream=s, **win)
    gk, gv = bt.pool.gather(0, moved[0], totals[0], stream=s)[:2]
    s.synchronize()
    assert bt.pool.check() == 0
    assert torch.equal(dec, want)
    for b, n in enumerate(totals):
        ref = attend(q[b:b + 1].cpu(), held(bt.k[b], kv), held(bt.v[b], kv), torch.tensor([n - 1]), window, 2 if window else 0)
        check(pre[b:b + 1], *ref, io, kv, f"prefill {b}")
    for got, rows in ((gk, bt.k[0]), (gv, bt.v[0])):
        assert torch.equal(got.view(bt.dt).transpose(0, 1).cpu().double(), held(rows, kv))
