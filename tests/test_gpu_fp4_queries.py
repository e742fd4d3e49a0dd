"""Queries over 4-bit pools hold over their whole type: bf16 rows beyond f16's range, either way.

The pages are attended in f16, so a bf16 row is brought into f16's range by a power of two that its scores are multiplied by
again.  Tolerances: tests/paged_cases.py.  A row that goes as it is (largest element at least 2^-1) has elements off by up to
2^-25; over 128 elements and keys of magnitude about 1 that is 128 * 2^-25 / sqrt(128) = 2^-21.5 of a score, inside the
2^-14 that c = 2^-13 has to spare.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from tests.paged_cases import Batch, attend, check, held  # noqa: E402

pytestmark = pytest.mark.gpu

LENS = [1, 17, 100, 700]
SHAPES = [(128, 28, 4), (128, 16, 1), (64, 14, 2), (64, 12, 1)]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def times(q, e):
    """q * 2^e, exactly (2^e may be past the type's own powers in one step)."""
    h = e // 2
    return (q.float() * 2.0 ** h * 2.0 ** (e - h)).to(q.dtype)


def refs(bt, q, pos, window, scale):
    r = [attend(q[b], held(bt.k[b], "fp4"), held(bt.v[b], "fp4"), pos[b], window, 0, scale=scale) for b in range(bt.B)]
    return r


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("e", [17, 40, 100, -10, -40, -100])
@pytest.mark.parametrize("D,Hq,Hkv", SHAPES)
def test_decode(D, Hq, Hkv, e, window):
    bt = Batch(D + Hq, "fp4", "bf16", D, Hq, Hkv, LENS).fill()
    q = times(bt.rows(bt.B, Hq), e)
    scale = 2.0 ** -e / math.sqrt(D)
    out = torch.full_like(q, 7.0).to(bt.dev)
    bt.pool.paged_decode(0, q.to(bt.dev), bt.device_table(), bt.lens(), out, scale=scale, window=window)
    assert bt.pool.check() == 0
    for b, r in enumerate(refs(bt, q[:, None], [torch.tensor([n - 1]) for n in LENS], window, scale)):
        check(out[b:b + 1], *r, "bf16", "fp4", f"sequence {b}")


CHUNKS = [(0, 1), (37, 100), (3000, 9)]


@pytest.mark.parametrize("chunks", [CHUNKS, [(3000, 9)]], ids=["3", "1"])
@pytest.mark.parametrize("e,window", [(17, 0), (40, 50), (100, 0), (-10, 0), (-40, 0), (-100, 50)])
@pytest.mark.parametrize("D,Hq,Hkv", SHAPES)
def test_prefill(D, Hq, Hkv, e, window, chunks):
    """Whole and split (the last chunk alone) tiles."""
    bt = Batch(D + Hq, "fp4", "bf16", D, Hq, Hkv, [a + n for a, n in chunks]).fill()
    q = [times(bt.rows(n, Hq), e) for _, n in chunks]
    scale = 2.0 ** -e / math.sqrt(D)
    cu = torch.tensor([0] + [n for _, n in chunks]).cumsum(0).int().to(bt.dev)
    start = torch.tensor([a for a, _ in chunks], dtype=torch.int32, device=bt.dev)
    qd = torch.cat(q).to(bt.dev)
    out = torch.full_like(qd, 7.0)
    bt.pool.paged_prefill(0, qd, cu, start, bt.device_table(), out, scale=scale, window=window)
    assert bt.pool.check() == 0
    for b, r in enumerate(refs(bt, q, [torch.arange(a, a + n) for a, n in chunks], window, scale)):
        check(out[int(cu[b]):int(cu[b + 1])], *r, "bf16", "fp4", f"chunk {b}")


@pytest.mark.parametrize("D,Hq,Hkv", SHAPES)
def test_rows_of_different_magnitudes(D, Hq, Hkv):
    """Heads and tokens side by side, 2^-40 to 2^17 (the scale makes the largest ordinary); infinities stay in their rows."""
    bt = Batch(D, "fp4", "bf16", D, Hq, Hkv, LENS).fill()
    q = bt.rows(bt.B, Hq)
    es = [17, 0, -40, 16, 15, -1, 12]
    for b in range(bt.B):
        for h in range(Hq):
            q[b, h] = times(q[b, h], es[(h + b) % len(es)])
    scale = 2.0 ** -17 / math.sqrt(D)
    ref = refs(bt, q[:, None], [torch.tensor([n - 1]) for n in LENS], 0, scale)
    bad = q.clone()
    bad[1, Hq - 1, 3], bad[2, 0, 5] = math.inf, math.nan
    for poisoned in (False, True):
        qd = (bad if poisoned else q).to(bt.dev)
        dec, pre = torch.full_like(qd, 7.0), torch.full_like(qd, 7.0)
        bt.pool.paged_decode(0, qd, bt.device_table(), bt.lens(), dec, scale=scale)
        cu = torch.arange(bt.B + 1, dtype=torch.int32, device=bt.dev)
        bt.pool.paged_prefill(0, qd, cu, bt.lens() - 1, bt.device_table(), pre, scale=scale)
        assert bt.pool.check() == 0
        for got in (dec, pre):
            if poisoned:
                assert got[1, Hq - 1].isnan().all() and got[2, 0].isnan().all()
                got[1, Hq - 1], got[2, 0] = ref[1][0][0, Hq - 1].to(got), ref[2][0][0, 0].to(got)
            for b, r in enumerate(ref):
                check(got[b:b + 1], *r, "bf16", "fp4", f"sequence {b}")


@pytest.mark.parametrize("D,Hq,Hkv", SHAPES[:3])
def test_rotated_rows(D, Hq, Hkv):
    """Rotation commutes with powers of two, so rows that all need a factor give the same bits, and an ordinary row the same
    within both tolerances."""
    bt = Batch(D, "fp4", "bf16", D, Hq, Hkv, LENS).fill()
    q = bt.rows(bt.B, Hq)
    got = {}
    for e in (0, 20, 60, -20):
        qd, scale = times(q, e).to(bt.dev), 2.0 ** -e / math.sqrt(D)
        dec, pre = torch.zeros_like(qd), torch.zeros_like(qd)
        bt.pool.paged_decode(0, qd, bt.device_table(), bt.lens(), dec, scale=scale, rope_theta=1e4)
        cu = torch.arange(bt.B + 1, dtype=torch.int32, device=bt.dev)
        bt.pool.paged_prefill(0, qd, cu, bt.lens() - 1, bt.device_table(), pre, scale=scale, rope_theta=1e4)
        assert bt.pool.check() == 0
        got[e] = (dec, pre)
    most = max(held(x, "fp4").abs().max().item() for x in bt.v)            # A, and F over its mass of at least 1, are at most
    for i in range(2):
        assert torch.equal(got[20][i], got[60][i]) and torch.equal(got[20][i], got[-20][i])
        x, y = got[0][i].double(), got[20][i].double()
        tol = 2 * (2.0 ** -8 * 1.01 * (x.abs() + 2.0 ** -8 * most) + (2.0 ** -11 + 2.0 ** -13) * most + 2.0 ** -25 * max(LENS) * most)
        assert ((x - y).abs() <= tol).all()


def test_small_rows_by_powers_of_two():
    """Rows below the format's scales, held as a user can: multiplied by a power of two on the way in, the softmax scale and the
    outputs divided by it.  The same bits as the rows at their ordinary size give."""
    ordinary = Batch(5, "fp4", "bf16", 128, 8, 2, LENS).fill()
    small = Batch(5, "fp4", "bf16", 128, 8, 2, LENS)
    k, v = [times(x, -9) for x in small.k], [times(x, -12) for x in small.v]           # the model's rows
    assert (held(v[3], "fp4") == 0).all() and (held(k[3], "fp4") == 0).float().mean() > 0.5
    small.k, small.v = [times(x, 9) for x in k], [times(x, 12) for x in v]             # what is appended
    small.fill()
    q = ordinary.rows(4, 8).to(ordinary.dev)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    ordinary.pool.paged_decode(0, q, ordinary.device_table(), ordinary.lens(), a)
    small.pool.paged_decode(0, q, small.device_table(), small.lens(), b, scale=1 / math.sqrt(128))
    assert ordinary.pool.check() == small.pool.check() == 0
    assert torch.equal(times(a, -12), times(b, -12))
    r = refs(small, q.cpu()[:, None], [torch.tensor([n - 1]) for n in LENS], 0, 1 / math.sqrt(128))
    for i in range(4):
        check(b[i:i + 1], *r[i], "bf16", "fp4", f"sequence {i}")
