"""The 4-bit pool: append, gather, block copy, decode and prefill against the codec's definition in 64 bits.

Pages are compared for equality (the codec is exact in its definition), attention within the tolerance derived in
tests/paged_cases.py over the values that the pool holds.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from tests.paged_cases import Batch, attend, check, held  # noqa: E402

pytestmark = pytest.mark.gpu

LENS = [1, 2, 15, 16, 17, 33, 100, 257, 600, 1000]
SHAPES = [("bf16", 128, 28, 4), ("f16", 128, 8, 8), ("bf16", 64, 14, 2), ("f16", 64, 16, 1), ("bf16", 128, 12, 1),
          ("bf16", 128, 1, 1), ("f16", 64, 9, 3)]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def values(bt, layer=0):
    """The values of every sequence, [K, V] per sequence, [n][Hkv][D] on the CPU."""
    r = []
    for b, n in enumerate(bt.totals):
        k, v = bt.pool.gather(layer, bt.device_table()[b], n)[:2]
        assert k.dtype == v.dtype == bt.dt
        r.append([x.transpose(0, 1).cpu() for x in (k, v)])
    return r


def same_as_held(bt, layer=0):
    for b, (k, v) in enumerate(values(bt, layer)):
        assert torch.equal(k.double(), held(bt.k[b], "fp4")) and torch.equal(v.double(), held(bt.v[b], "fp4")), b


def decode_ref(bt, q, scale=None):
    r = [attend(q[b:b + 1].cpu(), held(bt.k[b], "fp4"), held(bt.v[b], "fp4"), torch.tensor([n - 1]), scale=scale)
         for b, n in enumerate(bt.totals)]
    return tuple(torch.cat(x) for x in zip(*r))


@pytest.mark.parametrize("io,D", [("bf16", 128), ("f16", 64), ("f16", 128), ("bf16", 64)])
def test_append_holds_the_definition(io, D):
    """Every magnitude the io type has: normal rows, outliers, ties between codes, groups of zeros, groups whose scale rounds
    to 0 or is subnormal, values beyond the largest scale, infinities."""
    bt = Batch(1, "fp4", io, D, 2, 2, [517])
    for x in (bt.k[0], bt.v[0]):
        x[10:60] *= 2.0 ** torch.arange(-25, 25).clamp(-25, 14).double()[:, None, None].to(x.dtype)
        x[60:70] = 0.0
        x[70:80, :, ::16] = 0.0
        x[80:90] = -0.0
        x[90] = torch.finfo(x.dtype).max
        x[91] = torch.finfo(x.dtype).tiny
        x[92, :, 3::16] = math.inf
        x[93, :, 5::16] = -math.inf
        # every border between codes, exactly, under scales 1, 1.125, 2^-9 and 448 (the element of 6 scales sets it)
        half = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, 0.0])
        for i, sc in enumerate((1.0, 1.125, 2.0 ** -9, 448.0)):
            x[94 + i] = (half * sc).repeat(D // 16).to(x.dtype)
        x[100:200] = (x[100:200].float() * 4).round().to(x.dtype) / 4
    bt.fill()
    assert bt.pool.check() == 0
    same_as_held(bt)


def test_append_skips_and_flags():
    from voidweb_b200 import _lib as C
    bt = Batch(2, "fp4", "bf16", 128, 2, 2, [40]).fill()
    before = bt.pool.pages_u8().clone()
    k, v = bt.rows(3, 2).to(bt.dev), bt.rows(3, 2).to(bt.dev)
    bt.pool.append(0, k, v, torch.tensor([-1, bt.nb * 16, -5], device=bt.dev))
    assert bt.pool.check() == C.VW_DEV_ERR_SLOT
    assert torch.equal(before, bt.pool.pages_u8())
    bt.pool.append(0, k, v, torch.full((3,), -1, device=bt.dev))
    bt.pool.append(0, k[:0], v[:0], torch.zeros(0, dtype=torch.int64, device=bt.dev))
    assert bt.pool.check() == 0
    for bad in ((k.float(), v, 8), (k, v.cpu(), 8), (k[:, :, ::2], v, 8), (k.transpose(0, 1), v, 8), (k, v, 4)):
        with pytest.raises(ValueError):
            bt.pool.append(0, bad[0], bad[1], torch.zeros(3, dtype=torch.int64 if bad[2] == 8 else torch.int32, device=bt.dev))


@pytest.mark.parametrize("io,D,Hq,Hkv", SHAPES)
@pytest.mark.parametrize("scale", [0.0, 0.25])
def test_decode(io, D, Hq, Hkv, scale):
    bt = Batch(D + Hq, "fp4", io, D, Hq, Hkv, LENS).fill()
    q = bt.rows(bt.B, Hq).to(bt.dev)
    out = torch.full_like(q, 7.0)
    bt.pool.paged_decode(0, q, bt.device_table(), bt.lens(), out, scale=scale)
    assert bt.pool.check() == 0
    check(out, *decode_ref(bt, q, scale or None), io, "fp4")


@pytest.mark.parametrize("io,D,Hq,Hkv", [SHAPES[0], SHAPES[3]])
def test_decode_split_over_the_grid(io, D, Hq, Hkv):
    for totals in ([30011, 9000], [300 + 7 * i for i in range(67)], [1] * 130):
        bt = Batch(7, "fp4", io, D, Hq, Hkv, totals).fill()
        q = bt.rows(bt.B, Hq).to(bt.dev)
        out = torch.zeros_like(q)
        bt.pool.paged_decode(0, q, bt.device_table(), bt.lens(), out)
        assert bt.pool.check() == 0
        check(out, *decode_ref(bt, q), io, "fp4")


def test_peaked_and_wide_scores():
    """Keys with large channels (one key takes nearly all) and rows of widely different magnitudes."""
    bt = Batch(9, "fp4", "bf16", 128, 8, 2, [333, 700])
    for x in bt.k:
        x[:, :, 5] *= 30
        x *= 2.0 ** (torch.arange(len(x)) % 9 - 4).to(x.dtype)[:, None, None]
    for x in bt.v:
        x *= 2.0 ** (torch.arange(len(x)) % 21 - 10).to(x.dtype)[:, None, None]
    bt.fill()
    q = bt.rows(2, 8).to(bt.dev)
    out = torch.zeros_like(q)
    bt.pool.paged_decode(0, q, bt.device_table(), bt.lens(), out)
    # scores here reach 30 * 16 * 3: rows of |s| up to S put S * 128 * 2^-24 on a score, and as much on p
    ref, A, F = decode_ref(bt, q)
    S = max((q[b].cpu().double().abs() @ held(bt.k[b], "fp4").abs().amax((0, 1))).max().item() / math.sqrt(128) for b in range(2))
    got = out.cpu().double()
    tol = 2.0 ** -8 * 1.01 * ref.abs() + (2.0 ** -11 + 2.0 ** -13 + 2 * S * 2.0 ** -20) * A + 2.0 ** -25 * F
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("io,D,Hq,Hkv", [SHAPES[0], SHAPES[1], SHAPES[2], SHAPES[4]])
def test_fused_append_is_append_then_decode(io, D, Hq, Hkv):
    """Outputs and pages, bit for bit; over layers launched as programmatic dependents, planned, in fixed scratch, and in a
    replayed graph."""
    from voidweb_b200 import _lib as C
    L = 3
    a = Batch(4, "fp4", io, D, Hq, Hkv, LENS, layers=L).fill([n - 1 for n in LENS])
    b = Batch(4, "fp4", io, D, Hq, Hkv, LENS, layers=L).fill()
    q = [a.rows(a.B, Hq).to(a.dev) for _ in range(L)]
    kn, vn = (torch.stack([x[-1] for x in y]).to(a.dev) for y in (a.k, a.v))
    table, lens = a.device_table(), a.lens()
    oa, ob = ([torch.zeros_like(x) for x in q] for _ in range(2))
    for l in range(L):
        b.pool.paged_decode(l, q[l], table, lens, ob[l])
        a.pool.paged_decode(l, q[l], table, lens, oa[l], k_new=kn, v_new=vn,
                            flags=C.VW_DECODE_PDL | C.VW_DECODE_EARLY_PAGES if l else 0)
    assert a.pool.check() == b.pool.check() == 0
    assert all(torch.equal(x, y) for x, y in zip(oa, ob))
    assert torch.equal(a.pool.pages_u8(), b.pool.pages_u8())
    same_as_held(a, L - 1)
    a.pool.plan(table, lens, Hq)
    o = torch.zeros_like(q[0])
    a.pool.paged_decode(0, q[0], table, lens, o, k_new=kn, v_new=vn, flags=C.VW_DECODE_PLANNED)
    assert a.pool.check() == 0 and torch.equal(o, oa[0])
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    o.zero_()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        a.pool.paged_decode(0, q[0], table, lens, o, k_new=kn, v_new=vn)
    g.replay()
    assert a.pool.check() == 0 and torch.equal(o, oa[0])


def test_rope_rotates_before_it_quantises():
    """A rotated fused append leaves what appending the rotated rows leaves, and the decode is that of rotated queries."""
    from tests.test_gpu_window import device_rope
    lens, theta = [1, 20, 300], 1e6
    for io, D in (("bf16", 128), ("f16", 64)):
        a = Batch(6, "fp4", io, D, 8, 2, lens).fill([n - 1 for n in lens])
        b = Batch(6, "fp4", io, D, 8, 2, lens).fill([n - 1 for n in lens])
        q = a.rows(3, 8).to(a.dev)
        kn, vn = (torch.stack([x[-1] for x in y]).to(a.dev) for y in (a.k, a.v))
        oa, ob = torch.zeros_like(q), torch.zeros_like(q)
        a.pool.paged_decode(0, q, a.device_table(), a.lens(), oa, k_new=kn, v_new=vn, rope_theta=theta)
        b.pool.paged_decode(0, device_rope(q, lens, theta), b.device_table(), b.lens(), ob, k_new=device_rope(kn, lens, theta),
                            v_new=vn)
        assert a.pool.check() == b.pool.check() == 0
        assert torch.equal(oa, ob) and torch.equal(a.pool.pages_u8(), b.pool.pages_u8())


PREFILLS = [[(0, 1)], [(0, 64), (37, 100), (500, 7), (0, 1), (1000, 300)], [(123, 65), (0, 129)], [(0, 200), (300, 0), (7, 63)]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("chunks", PREFILLS, ids=[str(len(c)) for c in PREFILLS])
@pytest.mark.parametrize("io,D,Hq,Hkv", SHAPES)
def test_prefill(io, D, Hq, Hkv, chunks, causal):
    totals = [a + n for a, n in chunks]
    bt = Batch(len(chunks) + D, "fp4", io, D, Hq, Hkv, totals).fill([a for a, _ in chunks])
    q = [bt.rows(n, Hq) for _, n in chunks]
    cu = torch.tensor([0] + [n for _, n in chunks]).cumsum(0).int().to(bt.dev)
    start = torch.tensor([a for a, _ in chunks], dtype=torch.int32, device=bt.dev)
    kn = torch.cat([x[a:] for x, (a, _) in zip(bt.k, chunks)]).to(bt.dev)
    vn = torch.cat([x[a:] for x, (a, _) in zip(bt.v, chunks)]).to(bt.dev)
    qd = torch.cat(q + [bt.rows(3, Hq)]).to(bt.dev)          # rows behind the last chunk stay as they were
    kn, vn = (torch.cat((x, torch.zeros(3, Hkv, D, dtype=bt.dt, device=bt.dev))) for x in (kn, vn))
    out = torch.full_like(qd, 7.0)
    bt.pool.paged_prefill(0, qd, cu, start, bt.device_table(), out, k_new=kn, v_new=vn, causal=causal)
    assert bt.pool.check() == 0
    same_as_held(bt)
    for b, (a, n) in enumerate(chunks):
        if n:
            ref = attend(q[b], held(bt.k[b], "fp4"), held(bt.v[b], "fp4"), torch.arange(a, a + n), causal=causal)
            check(out[int(cu[b]):int(cu[b + 1])], *ref, io, "fp4", f"chunk {b}")
    assert (out[-3:] == 7.0).all()


def test_prompt_then_steps_then_fork():
    """Used together: a prompt in two chunks, decodes that append, the last page forked copy-on-write, both branches continued,
    and the caches read back."""
    n, forks = 400, 12
    bt = Batch(12, "fp4", "bf16", 128, 14, 2, [n, n + forks], layers=2)
    bt.k[1][:n], bt.v[1][:n] = bt.k[0], bt.v[0]
    full, half = (n - 1) // 16, bt.table[0, (n - 1) // 16].item()
    bt.table[1, :full + 1] = bt.table[0, :full + 1]           # sequence 1 starts as a fork of sequence 0
    q = bt.rows(n, 14)
    qd, kd, vd = q.to(bt.dev), bt.k[0].to(bt.dev), bt.v[0].to(bt.dev)
    out = torch.zeros_like(qd)

    def i32(*x):
        return torch.tensor(x, dtype=torch.int32, device=bt.dev)

    at = 0
    for m in (260, 137):
        for l in range(2):
            bt.pool.paged_prefill(l, qd[at:at + m], i32(0, m), i32(at), bt.device_table()[:1], out[at:at + m],
                                  k_new=kd[at:at + m], v_new=vd[at:at + m])
        at += m
    for p in range(at, n):
        for l in range(2):
            bt.pool.paged_decode(l, qd[p:p + 1], bt.device_table()[:1], i32(p + 1), out[p:p + 1], k_new=kd[p:p + 1],
                                 v_new=vd[p:p + 1])
    check(out, *attend(q, held(bt.k[0], "fp4"), held(bt.v[0], "fp4"), torch.arange(n)), "bf16", "fp4")
    free = (set(range(bt.nb)) - set(bt.table.flatten().tolist()))
    fresh = sorted(free)[0]
    if n % 16:
        bt.pool.block_copy(torch.tensor([[half, fresh]], dtype=torch.int32, device=bt.dev))
        bt.table[1, full] = fresh
    for p in range(n, n + forks):
        qq = bt.rows(1, 14)
        o = torch.zeros_like(qq).to(bt.dev)
        kn, vn = bt.k[1][p:p + 1].to(bt.dev), bt.v[1][p:p + 1].to(bt.dev)
        for l in range(2):
            bt.pool.paged_decode(l, qq.to(bt.dev), bt.device_table()[1:], i32(p + 1), o, k_new=kn, v_new=vn)
        ref = attend(qq, held(bt.k[1][:p + 1], "fp4"), held(bt.v[1][:p + 1], "fp4"), torch.tensor([p]))
        check(o, *ref, "bf16", "fp4", f"token {p}")
    assert bt.pool.check() == 0
    for l in range(2):
        same_as_held(bt, l)


def test_block_copy_moves_whole_records():
    for D, Hkv, L in ((128, 3, 2), (64, 1, 3)):
        bt = Batch(3, "fp4", "f16", D, Hkv, Hkv, [50, 70], layers=L, spare=9).fill()
        used = set(bt.table.flatten().tolist())
        free = [i for i in range(bt.nb) if i not in used]
        pairs = [(bt.table[0, 0].item(), free[0]), (bt.table[1, 2].item(), free[1])]
        before = bt.pool.pages_u8().clone().view(L, bt.nb, -1)
        bt.pool.block_copy(torch.tensor(pairs, dtype=torch.int32, device=bt.dev))
        after = bt.pool.pages_u8().view(L, bt.nb, -1)
        for s, d in pairs:
            before[:, d] = before[:, s]
        assert bt.pool.check() == 0 and torch.equal(before, after)


def test_bad_pages_are_flagged_and_hold_zeros():
    """A block id outside the pool reads as zero keys and values in decode and prefill; the others' outputs are right."""
    from voidweb_b200 import _lib as C
    bt = Batch(5, "fp4", "bf16", 128, 4, 1, [40, 40]).fill()
    table = bt.device_table()
    table[0, 1] = bt.nb
    bt.k[0][16:32] = 0
    bt.v[0][16:32] = 0
    q = bt.rows(2, 4).to(bt.dev)
    out = torch.zeros_like(q)
    bt.pool.paged_decode(0, q, table, bt.lens(), out)
    assert bt.pool.check() == C.VW_DEV_ERR_BLOCK_ID
    check(out, *decode_ref(bt, q), "bf16", "fp4")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=bt.dev)  # noqa: E731
    bt.pool.paged_prefill(0, q, i32(0, 1, 2), i32(39, 39), table, out)
    assert bt.pool.check() == C.VW_DEV_ERR_BLOCK_ID
    check(out, *decode_ref(bt, q), "bf16", "fp4")
    k, v = bt.pool.gather(0, table[0], 40)[:2]
    assert bt.pool.check() == C.VW_DEV_ERR_BLOCK_ID
    assert torch.equal(k[:, 32:].transpose(0, 1).cpu().double(), held(bt.k[0], "fp4")[32:])
    bt.pool.append(0, q[:, :1].contiguous(), q[:, :1].contiguous(), torch.tensor([5, -1], device=bt.dev))
    assert bt.pool.check() == 0


def test_host_step_and_forward_buffers():
    L = 3
    bt = Batch(6, "fp4", "bf16", 128, 8, 2, [5, 100, 400], layers=L).fill([4, 99, 399])
    q = torch.stack([bt.rows(3, 8) for _ in range(L)]).pin_memory()
    kn = torch.stack([torch.stack([x[-1] for x in bt.k])] * L).pin_memory()
    vn = torch.stack([torch.stack([x[-1] for x in bt.v])] * L).pin_memory()
    table, lens = bt.device_table().cpu().pin_memory(), bt.lens().cpu().pin_memory()
    out = torch.zeros_like(q).pin_memory()
    for _ in range(3):                                  # direct, recorded, replayed
        out.zero_()
        bt.pool.decode_step_host(q, kn, vn, table, lens, out)
        for l in range(L):
            check(out[l], *decode_ref(bt, q[l]), "bf16", "fp4", f"layer {l}")
    assert bt.pool.check() == 0


def test_fixed_scratch_and_caller_owned_pages():
    import ctypes
    from voidweb_b200 import _lib as C
    from voidweb_b200.kv import KvPool, PoolSpec, _ptr, _stream
    bt = Batch(8, "fp4", "bf16", 128, 8, 2, [3000, 17, 900]).fill()
    spec = PoolSpec(1, 2, 128, bt.nb, kv_dtype="fp4", io_dtype="bf16", max_batch=4)
    assert spec.block_bytes * bt.nb == bt.pool.data_bytes and bt.pool.scale_bytes == 0 and bt.pool.scales_f32() is None
    mine = torch.zeros(bt.pool.data_bytes, dtype=torch.uint8, device=bt.dev)
    pool = KvPool(spec, data=mine)
    mine.copy_(bt.pool.pages_u8())
    q, table, lens = bt.rows(3, 8).to(bt.dev), bt.device_table(), bt.lens()
    a, b, c = (torch.zeros_like(q) for _ in range(3))
    bt.pool.paged_decode(0, q, table, lens, a)
    pool.paged_decode(0, q, table, lens, b)
    args = C.DecodeArgs(0, 3, 8, table.shape[1], _ptr(q), _ptr(table), _ptr(lens), _ptr(c), None, None, 0.0, 0, 0.0, 0)
    C.check(C.lib().vw_paged_decode_static(pool.handle, ctypes.byref(args), _stream()))
    assert pool.check() == 0 and torch.equal(a, b) and torch.equal(a, c)
    check(a, *decode_ref(bt, q), "bf16", "fp4")


def test_wait_that_runs_out_is_an_error_and_the_pool_recovers():
    from voidweb_b200 import _lib as C
    bt = Batch(14, "fp4", "bf16", 128, 8, 2, [500, 60]).fill()
    q, table, lens = bt.rows(2, 8).to(bt.dev), bt.device_table(), bt.lens()
    out = torch.zeros_like(q)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=bt.dev)  # noqa: E731
    bt.pool.set_wait_limit(20000)
    bt.pool.paged_decode(0, q, table, lens, out)       # waits for nothing but its own loads
    assert bt.pool.check() == 0
    check(out, *decode_ref(bt, q), "bf16", "fp4")
    bt.pool.paged_prefill(0, q, i32(0, 1, 2), lens - 1, table, out)
    assert bt.pool.check() & C.VW_DEV_ERR_TIMEOUT
    bt.pool.set_wait_limit(0)
    bt.pool.paged_decode(0, q, table, lens, out)
    assert bt.pool.check() == 0
    check(out, *decode_ref(bt, q), "bf16", "fp4")


def test_refusals():
    bt = Batch(10, "fp4", "bf16", 128, 8, 2, [100]).fill()
    q, lens, table = bt.rows(1, 8).to(bt.dev), bt.lens(), bt.device_table()
    out = torch.zeros_like(q)
    for a in ((q.float(), table, lens, out), (q, table.long(), lens, out), (q, table, lens.long(), out), (q, table, lens, out[:, :4]),
              (q[:, :, :64], table, lens, out), (q, table, lens[:0], out)):
        with pytest.raises(ValueError):
            bt.pool.paged_decode(0, *a)
    with pytest.raises(ValueError):
        bt.pool.gather(0, table[0], table.shape[1] * 16 + 1)
    assert bt.pool.check() == 0


@pytest.mark.parametrize("kv,io,D,Hq,Hkv,window,sinks", [
    ("fp4", "bf16", 128, 28, 4, 0, 0), ("fp4", "f16", 64, 16, 1, 0, 0), ("fp4", "f16", 128, 8, 8, 3000, 7),
    ("bf16", "bf16", 128, 28, 4, 4000, 4), ("f16", "f16", 64, 6, 2, 2000, 40), ("bf16", "bf16", 128, 3, 1, 100000, 0)])
@pytest.mark.parametrize("chunks", [[(6000, 5)], [(3001, 1), (100, 40)], [(8000, 33), (0, 9), (15, 1), (2000, 130)]],
                         ids=["1", "2", "4"])
def test_few_queries_over_long_contexts(kv, io, D, Hq, Hkv, window, sinks, chunks):
    """The keys of a tile split over several CTAs and merged; decodes around it on the same stream share the scratch."""
    from tests.paged_cases import v_scales
    totals = [a + n for a, n in chunks]
    bt = Batch(len(chunks) + D, kv, io, D, Hq, Hkv, totals).fill()
    q = [bt.rows(n, Hq) for _, n in chunks]
    cu = torch.tensor([0] + [n for _, n in chunks]).cumsum(0).int().to(bt.dev)
    start = torch.tensor([a for a, _ in chunks], dtype=torch.int32, device=bt.dev)
    qd = torch.cat(q).to(bt.dev)
    out, dec, table = torch.full_like(qd, 7.0), [], bt.device_table()
    last = torch.stack([x[-1] for x in q]).to(bt.dev)
    for _ in range(2):
        d = torch.zeros_like(last)
        bt.pool.paged_decode(0, last, table, bt.lens(), d, window=window, sinks=sinks)
        bt.pool.paged_prefill(0, qd, cu, start, table, out, window=window, sinks=sinks)
        dec.append(d)
    assert bt.pool.check() == 0
    assert torch.equal(dec[0], dec[1])
    for b, (a, n) in enumerate(chunks):
        ref = attend(q[b], held(bt.k[b], kv), held(bt.v[b], kv), torch.arange(a, a + n), window, sinks,
                     v_scale=v_scales(bt.v[b], kv))
        check(out[int(cu[b]):int(cu[b + 1])], *ref, io, kv, f"chunk {b}")
        check(dec[0][b:b + 1], *(x[-1:] for x in ref), io, kv, f"decode {b}")


@pytest.mark.parametrize("kv,window", [("fp4", 0), ("fp4", 5), ("bf16", 5)])
def test_largest_batch(kv, window):
    """1024 sequences (the most that a launch takes), decode and prefill, lengths 1 to 40."""
    totals = [1 + (7 * i) % 40 for i in range(1024)]
    bt = Batch(15, kv, "bf16", 64, 6, 2, totals, max_batch=1024).fill()
    q = bt.rows(1024, 6)
    out = torch.zeros_like(q).to(bt.dev)
    start, cu = bt.lens() - 1, torch.arange(1025, dtype=torch.int32, device=bt.dev)
    for f in ("decode", "prefill"):
        if f == "decode":
            bt.pool.paged_decode(0, q.to(bt.dev), bt.device_table(), bt.lens(), out, window=window, sinks=2 if window else 0)
        else:
            out.zero_()
            bt.pool.paged_prefill(0, q.to(bt.dev), cu, start, bt.device_table(), out, window=window, sinks=2 if window else 0)
        assert bt.pool.check() == 0
        for b in range(0, 1024, 37):
            ref = attend(q[b:b + 1], held(bt.k[b], kv), held(bt.v[b], kv), torch.tensor([totals[b] - 1]), window, 2 if window else 0)
            check(out[b:b + 1], *ref, "bf16", kv, f"{f} {b}")
    with pytest.raises(Exception):
        bt.pool.paged_decode(0, torch.zeros(1025, 6, 64, dtype=torch.bfloat16, device=bt.dev),
                             torch.zeros(1025, 3, dtype=torch.int32, device=bt.dev),
                             torch.ones(1025, dtype=torch.int32, device=bt.dev),
                             torch.zeros(1025, 6, 64, dtype=torch.bfloat16, device=bt.dev), window=window, sinks=2 if window else 0)


@pytest.mark.parametrize("kv,window", [("fp4", 0), ("f16", 70)])
def test_prefill_with_more_query_heads_than_rows_of_a_tile(kv, window):
    """71 and 200 query heads on one KV head: one token's rows span tiles."""
    for Hq in (71, 200):
        chunks = [(90, 3), (0, 5)]
        bt = Batch(Hq, kv, "f16", 64, Hq, 1, [a + n for a, n in chunks]).fill()
        q = [bt.rows(n, Hq) for _, n in chunks]
        cu = torch.tensor([0, 3, 8], dtype=torch.int32, device=bt.dev)
        start = torch.tensor([90, 0], dtype=torch.int32, device=bt.dev)
        out = torch.zeros(8, Hq, 64, dtype=torch.float16, device=bt.dev)
        bt.pool.paged_prefill(0, torch.cat(q).to(bt.dev), cu, start, bt.device_table(), out, window=window)
        assert bt.pool.check() == 0
        for b, (a, n) in enumerate(chunks):
            ref = attend(q[b], held(bt.k[b], kv), held(bt.v[b], kv), torch.arange(a, a + n), window)
            check(out[int(cu[b]):int(cu[b + 1])], *ref, "f16", kv, f"{Hq} {b}")


@pytest.mark.parametrize("kv,window", [("fp4", 0), ("fp4", 20), ("bf16", 20), ("bf16", 0)])
def test_lengths_and_chunks_outside_the_tables(kv, window):
    """Flagged; nothing is written for them; the other sequences are right."""
    from voidweb_b200 import _lib as C
    bt = Batch(16, kv, "bf16", 128, 8, 2, [100, 50, 300], stride_extra=0).fill()
    q, table = bt.rows(3, 8), bt.device_table()
    qd = q.to(bt.dev)
    refs = [attend(q[b:b + 1], held(bt.k[b], kv), held(bt.v[b], kv), torch.tensor([n - 1]), window) for b, n in enumerate(bt.totals)]
    for bad in (0, -5, 320 + 1, 2 ** 31 - 1, 2 ** 31 - 17):
        out = torch.full_like(qd, 7.0)
        bt.pool.paged_decode(0, qd, table, bt.lens([100, bad, 300]), out, window=window)
        assert bt.pool.check() & C.VW_DEV_ERR_SEQ_LEN
        for b in (0, 2):
            check(out[b:b + 1], *refs[b], "bf16", kv, f"len {bad}")
        assert bad > 0 or (out[1] == 7.0).all()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=bt.dev)  # noqa: E731
    for cu, start in ((i32(0, 1, 2, 9), i32(99, 49, 299)), (i32(0, 1, 2, 2 ** 31 - 1), i32(99, 49, 299)),
                      (i32(0, 1, 2, 3), i32(99, 49, 2 ** 31 - 2)), (i32(0, 1, 2, 3), i32(99, 49, -1))):
        out = torch.full_like(qd, 7.0)
        bt.pool.paged_prefill(0, qd, cu, start, table, out, window=window)
        assert bt.pool.check() & C.VW_DEV_ERR_SEQ_LEN
        for b in (0, 1):
            check(out[b:b + 1], *refs[b], "bf16", kv, f"chunk {b}")
        assert (out[2] == 7.0).all()


def test_forward_pass_over_a_4_bit_pool():
    """The engine's symbol: a prompt and decode steps through voidweb_forward_pass."""
    import ctypes
    import numpy as np
    from voidweb_b200 import _lib as C
    L, Hq, Hkv, D, n = 2, 8, 2, 128, 60
    bt = Batch(17, "fp4", "bf16", D, Hq, Hkv, [n], layers=L)
    lib, q = C.lib(), bt.rows(n, Hq)
    table = np.ascontiguousarray(bt.table[0, :4].numpy().astype(np.uint32))

    def step(first, count, prefill):
        hq = torch.stack([q[first:first + count]] * L).pin_memory()
        hk, hv = (torch.stack([x[0][first:first + count]] * L).pin_memory() for x in (bt.k, bt.v))
        ho = torch.zeros_like(hq).pin_memory()
        C.check(lib.vw_forward_bind(bt.pool.handle, hq.data_ptr(), hk.data_ptr(), hv.data_ptr(), ho.data_ptr()))
        toks = (ctypes.c_uint32 * count)()
        d = C.SeqDescriptor(7, ctypes.addressof(toks), count, table.ctypes.data, len(table), 1 if prefill else 0)
        a = C.ForwardArgs(ctypes.addressof(d), 1, Hq * D, Hq, Hkv, L, 100, D, 0.0, 0, None)
        assert lib.voidweb_forward_pass(ctypes.byref(a)) == 0, lib.vw_last_error()
        return ho

    lib.vw_forward_set_seq_len(7, 0)
    try:
        outs = [step(0, 57, True)] + [step(p, 1, False) for p in range(57, n)]
    finally:
        lib.vw_forward_release(7)
        lib.vw_forward_bind(None, None, None, None, None)
    assert bt.pool.check() == 0
    ref = attend(q, held(bt.k[0], "fp4"), held(bt.v[0], "fp4"), torch.arange(n))
    for l in range(L):
        check(torch.cat([o[l] for o in outs]), *ref, "bf16", "fp4", f"layer {l}")
        same_as_held(bt, l)


@pytest.mark.parametrize("kv,window,chunks", [("fp4", 0, [(300, 1216)]), ("fp4", 333, [(900, 1216)]),
                                              ("bf16", 333, [(900, 700), (0, 500), (77, 24)]),
                                              ("bf16", 40, [(900, 1290)])])
def test_prefill_of_more_tiles_than_are_resident(kv, window, chunks):
    """304 and more tiles of 128 rows over 8 KV heads, where the SMs hold 296 together."""
    bt = Batch(18, kv, "bf16", 128, 32, 8, [a + n for a, n in chunks]).fill()
    q = [bt.rows(n, 32) for _, n in chunks]
    ns = [n for _, n in chunks]
    cu = torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=bt.dev)
    start = torch.tensor([a for a, _ in chunks], dtype=torch.int32, device=bt.dev)
    out = torch.zeros(sum(ns), 32, 128, dtype=torch.bfloat16, device=bt.dev)
    bt.pool.paged_prefill(0, torch.cat(q).to(bt.dev), cu, start, bt.device_table(), out, window=window, sinks=3 if window else 0)
    assert bt.pool.check() == 0
    for b, (a, n) in enumerate(chunks):
        ref = attend(q[b], held(bt.k[b], kv), held(bt.v[b], kv), torch.arange(a, a + n), window, 3 if window else 0)
        check(out[int(cu[b]):int(cu[b + 1])], *ref, "bf16", kv, f"chunk {b}")


def test_other_types_are_refused():
    """Rows of the other 16-bit type, 16-bit floats for ids; bit patterns of the right size pass."""
    bt = Batch(19, "fp4", "bf16", 64, 4, 2, [20]).fill()
    pool, table, lens = bt.pool, bt.device_table(), bt.lens()
    q = bt.rows(1, 4).to(bt.dev)
    out = torch.empty_like(q)
    want = pool.paged_decode(0, q, table, lens, out).clone()
    for bad in (dict(q=q.half()), dict(q=q.float()), dict(out=out.half()), dict(seq_lens=lens.float()),
                dict(block_tables=table.float()), dict(seq_lens=lens.long())):
        args = dict(dict(q=q, block_tables=table, seq_lens=lens, out=out), **bad)
        with pytest.raises(ValueError):
            pool.paged_decode(0, args["q"], args["block_tables"], args["seq_lens"], args["out"])
        with pytest.raises(ValueError):
            pool.paged_decode(0, args["q"], args["block_tables"], args["seq_lens"], args["out"], window=3)
    k = bt.k[0][:1].to(bt.dev)
    slots = torch.zeros(1, dtype=torch.int64, device=bt.dev)
    for kk, vv, ss in ((k.half(), k, slots), (k, k.float(), slots), (k, k, slots.int()), (k, k, slots.double())):
        with pytest.raises(ValueError):
            pool.append(0, kk, vv, ss)
    got = torch.empty_like(out)
    pool.paged_decode(0, q.view(torch.int16), table.view(torch.uint32), lens, got.view(torch.int16))
    assert torch.equal(got, want)
    assert pool.check() == 0


@pytest.mark.parametrize("kv", ["fp4", "bf16"])
def test_block_table_rows_past_31_bits_are_refused(kv):
    """2^26 blocks are 2^30 tokens; one more is refused before a launch, by every call that takes a window or a 4-bit pool."""
    import ctypes
    from voidweb_b200 import _lib as C
    bt = Batch(20, kv, "bf16", 64, 4, 2, [20]).fill()
    table, lens, q = bt.device_table(), bt.lens(), bt.rows(1, 4).to(bt.dev)
    out, cu = torch.full_like(q, 7.0), torch.tensor([0, 1], dtype=torch.int32, device=bt.dev)
    ptr, h, win = (lambda t: ctypes.c_void_p(t.data_ptr())), bt.pool.handle, C.Window(5, 1)
    st = torch.cuda.current_stream().cuda_stream
    big = (1 << 26) + 1
    d = C.DecodeArgs(0, 1, 4, big, ptr(q), ptr(table), ptr(lens), ptr(out), None, None, 0.0, 0, 0.0, 0)
    p = C.PrefillArgs(0, 1, 1, 4, big, C.VW_PREFILL_CAUSAL, ptr(q), None, None, ptr(cu), ptr(lens - 1), ptr(table), ptr(out), 0.0, 0.0)
    bad = C.VW_ERR_INVALID_ARG
    assert C.lib().vw_paged_decode_window(h, ctypes.byref(d), ctypes.byref(win), st) == bad
    assert C.lib().vw_paged_prefill_window(h, ctypes.byref(p), ctypes.byref(win), st) == bad
    if kv == "fp4":
        assert C.lib().vw_paged_decode(h, ctypes.byref(d), st) == bad
        assert C.lib().vw_paged_decode_static(h, ctypes.byref(d), st) == bad
        assert C.lib().vw_paged_prefill(h, ctypes.byref(p), st) == bad
    torch.cuda.synchronize()
    assert bt.pool.check() == 0 and (out == 7.0).all()
