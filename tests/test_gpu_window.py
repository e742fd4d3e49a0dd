"""Sliding-window attention with sinks (decode and prefill) against 64 bits.

Tolerances: tests/paged_cases.py.  Hidden block-table entries hold 0xFFFFFFFF
(an id that would be flagged if it were read) and hidden tokens inside visited
pages hold Inf or NaN.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from tests.paged_cases import Batch, attend, check, held, hidden_pages, v_scales  # noqa: E402

pytestmark = pytest.mark.gpu

KINDS = [("bf16", "bf16", 128, 28, 4), ("f16", "f16", 64, 14, 2), ("fp8", "bf16", 128, 32, 8), ("fp8", "f16", 128, 24, 2),
         ("bf16", "bf16", 128, 16, 1), ("bf16", "bf16", 64, 3, 3), ("f16", "f16", 128, 12, 1), ("fp4", "bf16", 128, 28, 4),
         ("fp4", "f16", 64, 14, 2), ("fp4", "f16", 128, 16, 1)]
WINDOWS = [(1, 0), (1, 1), (16, 0), (17, 3), (100, 4), (33, 16), (64, 40), (5, 1000), (250, 17), (2 ** 32 - 1, 2 ** 32 - 1)]
LENS = [1, 2, 15, 16, 17, 33, 100, 257, 600, 1000]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def windowed(bt, window, sinks, value=math.nan):
    """Hide what a decode at the last token does not see: table entries and rows."""
    for b, n in enumerate(bt.totals):
        bt.overwrite(b, min(sinks, n), max(min(sinks, n), n - window), value)
    return bt.device_table(lambda b, pg: hidden_pages(bt.totals[b] - 1, bt.totals[b] - 1, window, sinks)(pg))


def decode_ref(bt, q, window, sinks, scale=None):
    r = [attend(q[b:b + 1].cpu(), held(bt.k[b], bt.kv), held(bt.v[b], bt.kv), torch.tensor([n - 1]), window, sinks, scale=scale,
                v_scale=v_scales(bt.v[b], bt.kv))
         for b, n in enumerate(bt.totals)]
    return tuple(torch.cat(x) for x in zip(*r))


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("kv,io,D,Hq,Hkv", KINDS)
def test_decode(kv, io, D, Hq, Hkv, window, sinks):
    bt = Batch(window % 97 + sinks % 89 + D, kv, io, D, Hq, Hkv, LENS).fill()
    table = windowed(bt, window, sinks, math.nan if window % 2 else math.inf)
    q = bt.rows(bt.B, Hq).to(bt.dev)
    out = torch.full_like(q, 7.0)
    bt.pool.paged_decode(0, q, table, bt.lens(), out, window=window, sinks=sinks)
    assert bt.pool.check() == 0
    check(out, *decode_ref(bt, q, window, sinks), io, kv, f"window {window} sinks {sinks}")


@pytest.mark.parametrize("kv,io,D,Hq,Hkv", KINDS[:4] + KINDS[7:9])
def test_window_of_the_whole_context_is_the_plain_decode(kv, io, D, Hq, Hkv):
    bt = Batch(3, kv, io, D, Hq, Hkv, LENS + [4000]).fill()
    q = bt.rows(bt.B, Hq).to(bt.dev)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    bt.pool.paged_decode(0, q, bt.device_table(), bt.lens(), a)
    bt.pool.paged_decode(0, q, bt.device_table(), bt.lens(), b, window=4000)
    assert bt.pool.check() == 0
    assert torch.equal(a, b)


@pytest.mark.parametrize("kv,io,D,Hq,Hkv", [KINDS[0], KINDS[2], KINDS[7]])
def test_decode_split_over_the_grid(kv, io, D, Hq, Hkv):
    """Few long sequences (windows cut across many CTAs) and many short ones."""
    for totals, window, sinks in (([30011, 9000], 8190, 4), ([5000 + 37 * i for i in range(33)], 1000, 20)):
        bt = Batch(11, kv, io, D, Hq, Hkv, totals).fill()
        table = windowed(bt, window, sinks)
        q = bt.rows(bt.B, Hq).to(bt.dev)
        out = torch.zeros_like(q)
        bt.pool.paged_decode(0, q, table, bt.lens(), out, window=window, sinks=sinks)
        assert bt.pool.check() == 0
        check(out, *decode_ref(bt, q, window, sinks), io, kv)


def device_rope(rows, lens, theta):
    """rows [B][H][D] rotated at lens - 1 by the library: what a rotated append leaves in a scratch pool."""
    B, H, D = rows.shape
    io = "bf16" if rows.dtype == torch.bfloat16 else "f16"
    bt = Batch(1, io, io, D, H, H, lens)
    out = torch.zeros_like(rows)
    bt.pool.paged_decode(0, rows, bt.device_table(), bt.lens(), out, k_new=rows, v_new=rows, rope_theta=theta)
    got = [bt.pool.gather(0, bt.device_table()[b], n)[0][:, -1].view(rows.dtype) for b, n in enumerate(lens)]
    return torch.stack(got)


@pytest.mark.parametrize("kv,io,D,Hq,Hkv", [KINDS[0], KINDS[1], KINDS[2], KINDS[7], KINDS[8]])
def test_fused_append_rope_layers_and_graphs(kv, io, D, Hq, Hkv):
    """The step's rows appended by the decode, with and without rotation, over layers launched as programmatic dependents;
    then captured and replayed.  The rotated step equals the plain step over rows that the library rotated, bit for bit."""
    from voidweb_b200 import _lib as C
    window, sinks, L, theta = 40, 3, 3, 10000.0
    lens = LENS
    q0 = None
    outs = []
    for rotated in (True, False):
        bt = Batch(5, kv, io, D, Hq, Hkv, lens, layers=L).fill([n - 1 for n in lens])
        for b, n in enumerate(lens):
            bt.overwrite(b, min(sinks, n - 1), max(min(sinks, n - 1), n - window), math.nan)
        table = bt.device_table(lambda b, pg: hidden_pages(lens[b] - 1, lens[b] - 1, window, sinks)(pg))
        q0 = [bt.rows(bt.B, Hq).to(bt.dev) for _ in range(L)] if q0 is None else q0
        q = q0 if rotated else [device_rope(x, lens, theta) for x in q0]
        kn = torch.stack([x[-1] for x in bt.k]).to(bt.dev)
        kn = kn if rotated else device_rope(kn, lens, theta)
        vn = torch.stack([x[-1] for x in bt.v]).to(bt.dev)
        out = [torch.zeros_like(x) for x in q]
        dl = bt.lens()

        def step():
            for l in range(L):
                bt.pool.paged_decode(l, q[l], table, dl, out[l], k_new=kn, v_new=vn, window=window, sinks=sinks,
                                     rope_theta=theta if rotated else 0.0,
                                     flags=C.VW_DECODE_PDL | C.VW_DECODE_EARLY_PAGES if l else 0)

        step()
        assert bt.pool.check() == 0
        outs.append([x.clone() for x in out])
        if not rotated:
            for b in range(bt.B):
                bt.k[b][-1] = kn[b].cpu()
            for l in range(L):
                check(out[l], *decode_ref(bt, q[l], window, sinks), io, kv, f"layer {l}")
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            with torch.cuda.graph(g, stream=s):
                step()
        for x in out:
            x.zero_()
        torch.cuda.synchronize()
        g.replay()
        assert bt.pool.check() == 0
        assert all(torch.equal(a, b) for a, b in zip(outs[-1], out))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_step_host():
    window, sinks, L = 64, 4, 3
    bt = Batch(6, "bf16", "bf16", 128, 8, 2, [5, 100, 400], layers=L).fill([4, 99, 399])
    q = torch.stack([bt.rows(3, 8) for _ in range(L)]).pin_memory()
    kn = torch.stack([torch.stack([x[-1] for x in bt.k])] * L).pin_memory()
    vn = torch.stack([torch.stack([x[-1] for x in bt.v])] * L).pin_memory()
    table, lens = bt.device_table().cpu().pin_memory(), bt.lens().cpu().pin_memory()
    out = torch.zeros_like(q).pin_memory()
    for w in (window, window, window, 10 ** 6, 10 ** 6, window):     # direct, recorded, replayed; another window between
        out.zero_()
        bt.pool.decode_step_host(q, kn, vn, table, lens, out, window=w, sinks=sinks)
        for l in range(L):
            check(out[l], *decode_ref(bt, q[l], w, sinks), "bf16", "bf16", f"layer {l} window {w}")
    assert bt.pool.check() == 0


PREFILLS = [[(0, 1)], [(0, 5), (16, 16), (700, 130), (31, 1)], [(300, 257), (0, 129), (1000, 40)]]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 3), (100, 4), (64, 40), (5, 1000), (250, 17), (2 ** 32 - 1, 9)])
@pytest.mark.parametrize("chunks", PREFILLS, ids=[str(len(c)) for c in PREFILLS])
@pytest.mark.parametrize("kv,io,D,Hq,Hkv", KINDS)
def test_prefill(kv, io, D, Hq, Hkv, chunks, window, sinks):
    totals = [a + n for a, n in chunks]
    bt = Batch(len(chunks) + window % 31, kv, io, D, Hq, Hkv, totals).fill([a for a, _ in chunks])
    for b, (a, n) in enumerate(chunks):        # hidden from the whole chunk: NaN
        bt.overwrite(b, min(sinks, a), max(min(sinks, a), a + 1 - window), math.nan)
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
        ref = attend(q[b], held(bt.k[b], kv), held(bt.v[b], kv), torch.arange(a, a + n), window, sinks,
                     v_scale=v_scales(bt.v[b], kv))
        check(out[int(cu[b]):int(cu[b + 1])], *ref, io, kv, f"chunk {b}")


@pytest.mark.parametrize("kv,io,D,Hq,Hkv", KINDS[:4] + KINDS[7:9])
def test_prefill_whole_window_and_long_chunks(kv, io, D, Hq, Hkv):
    """A window of the whole context sees what a plain prefill sees; chunks of many tiles, the last rows ragged."""
    chunks = [(400, 300), (0, 40), (1000, 777)]
    bt = Batch(8, kv, io, D, Hq, Hkv, [a + n for a, n in chunks]).fill()
    q = bt.rows(1117, Hq).to(bt.dev)
    cu = torch.tensor([0, 300, 340, 1117], dtype=torch.int32, device=bt.dev)
    start = torch.tensor([a for a, _ in chunks], dtype=torch.int32, device=bt.dev)
    x, y = torch.zeros_like(q), torch.zeros_like(q)
    bt.pool.paged_prefill(0, q, cu, start, bt.device_table(), x)
    bt.pool.paged_prefill(0, q, cu, start, bt.device_table(), y, window=1777)
    assert bt.pool.check() == 0
    for b, (a, n) in enumerate(chunks):
        r = slice(int(cu[b]), int(cu[b + 1]))
        ref = attend(q[r].cpu(), held(bt.k[b], kv), held(bt.v[b], kv), torch.arange(a, a + n), v_scale=v_scales(bt.v[b], kv))
        check(x[r], *ref, io, kv, f"plain {b}")
        check(y[r], *ref, io, kv, f"window {b}")


def test_prefill_then_decode_steps():
    """Used together: a prompt in two windowed chunks, then decodes that append, with the blocks that left the window reused
    by nobody but poisoned; against one 64-bit pass over the whole sequence."""
    window, sinks, n = 48, 4, 420
    bt = Batch(21, "bf16", "bf16", 128, 14, 2, [n], layers=1)
    out = torch.zeros(n, 14, 128, dtype=torch.bfloat16, device=bt.dev)
    q = bt.rows(n, 14)
    qd, kd, vd = q.to(bt.dev), bt.k[0].to(bt.dev), bt.v[0].to(bt.dev)

    def i32(*x):
        return torch.tensor(x, dtype=torch.int32, device=bt.dev)

    at = 0
    for m in (260, 140):
        table = bt.device_table(lambda b, pg: hidden_pages(at, at + m - 1, window, sinks)(pg))
        bt.pool.paged_prefill(0, qd[at:at + m], i32(0, m), i32(at), table, out[at:at + m], k_new=kd[at:at + m],
                              v_new=vd[at:at + m], window=window, sinks=sinks)
        at += m
    for p in range(at, n):
        table = bt.device_table(lambda b, pg: hidden_pages(p, p, window, sinks)(pg))
        bt.pool.paged_decode(0, qd[p:p + 1], table, i32(p + 1), out[p:p + 1], k_new=kd[p:p + 1], v_new=vd[p:p + 1],
                             window=window, sinks=sinks)
    assert bt.pool.check() == 0
    check(out, *attend(q, held(bt.k[0], "bf16"), held(bt.v[0], "bf16"), torch.arange(n), window, sinks), "bf16", "bf16")


def test_lengths_that_are_refused_or_flagged():
    """seq_len 0 leaves its row; one beyond its table is flagged and ends; the other sequences are right."""
    from voidweb_b200 import _lib as C
    bt = Batch(9, "bf16", "bf16", 128, 8, 2, [100, 50, 300], stride_extra=0).fill()
    q = bt.rows(3, 8).to(bt.dev)
    out = torch.full_like(q, 7.0)
    bt.pool.paged_decode(0, q, bt.device_table(), bt.lens([100, 0, 300]), out, window=20, sinks=2)
    assert bt.pool.check() & C.VW_DEV_ERR_SEQ_LEN
    ref = decode_ref(bt, q, 20, 2)
    for b in (0, 2):
        check(out[b:b + 1], *(x[b:b + 1] for x in ref), "bf16", "bf16")
    assert (out[1] == 7.0).all()
    bt.pool.paged_decode(0, q, bt.device_table(), bt.lens([100, 50, 5000]), out, window=20, sinks=2)
    assert bt.pool.check() & C.VW_DEV_ERR_SEQ_LEN
    check(out[:2], *(x[:2] for x in ref), "bf16", "bf16")
    bt.pool.paged_decode(0, q[:0], bt.device_table()[:0], bt.lens()[:0], out[:0], window=20)
    assert bt.pool.check() == 0


def test_refusals():
    from voidweb_b200 import VoidwebError, _lib as C
    bt = Batch(10, "bf16", "bf16", 128, 8, 2, [100]).fill()
    q, lens, table = bt.rows(1, 8).to(bt.dev), bt.lens(), bt.device_table()
    out = torch.zeros_like(q)
    dec = bt.pool.paged_decode
    for bad in (dict(window=-1), dict(window=0, sinks=3), dict(window=4, sinks=-1), dict(window=2 ** 32)):
        with pytest.raises(ValueError):
            dec(0, q, table, lens, out, **bad)
    with pytest.raises(ValueError):
        dec(0, q.float(), table, lens, out, window=4)
    with pytest.raises(ValueError):
        dec(0, q, table.long(), lens, out, window=4)
    with pytest.raises(ValueError):
        dec(0, bt.rows(1, 16).to(bt.dev)[:, ::2], table, lens, out, window=4)
    with pytest.raises(ValueError):
        dec(0, q.cpu(), table, lens, out, window=4)
    bt.pool.plan(table, lens, 8)
    with pytest.raises(VoidwebError) as e:
        dec(0, q, table, lens, out, window=4, flags=C.VW_DECODE_PLANNED)
    assert e.value.code == C.VW_ERR_INVALID_ARG
    with pytest.raises(VoidwebError) as e:
        bt.pool.paged_prefill(0, q, torch.tensor([0, 1], dtype=torch.int32, device=bt.dev), lens, table, out, causal=False,
                              window=4)
    assert e.value.code == C.VW_ERR_INVALID_ARG
    assert bt.pool.check() == 0
