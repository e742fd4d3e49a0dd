"""Windows at the end of the longest block-table row that they take: 2^26 blocks, positions to 2^30.

Only the pages that a window or the sinks leave visible have blocks; every other entry of the row is an id outside the pool,
which would be flagged if it were read.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from tests.paged_cases import TYPES, attend, check, held, v_scales  # noqa: E402

pytestmark = pytest.mark.gpu

STRIDE = 1 << 26
WINDOW, SINKS = 150, 20


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.fixture(scope="module")
def table():
    return torch.full((2, STRIDE), -1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("kv,io,D,Hq,Hkv", [("fp4", "bf16", 128, 28, 4), ("fp4", "f16", 64, 16, 1), ("bf16", "bf16", 128, 28, 4),
                                            ("f16", "f16", 64, 6, 2), ("fp8", "bf16", 128, 16, 2)])
def test_last_positions(table, kv, io, D, Hq, Hkv, n):
    """Decode (n = 1, its row appended by the call) and prefill of the last n tokens of sequences of 2^30 and 2^30 - 21 tokens."""
    from voidweb_b200.kv import KvPool, PoolSpec
    g, dt, totals = torch.Generator().manual_seed(n + D), TYPES[io], [1 << 30, (1 << 30) - 21]
    kept = WINDOW + n + 16                            # tokens of the tail that have rows
    pool = KvPool(PoolSpec(1, Hkv, D, 64, kv_dtype=kv, io_dtype=io, fp8_mode="ocp", max_batch=2))
    pool.pages_u8().fill_(0xFF)
    if kv == "fp8":
        pool.scales_f32().fill_(math.nan)
    blocks, ks, vs = iter(torch.randperm(64, generator=g).tolist()), [], []
    table.fill_(-1)
    for b, total in enumerate(totals):
        first = total - kept
        for pg in list(range((SINKS + 15) // 16)) + list(range(first // 16, (total + 15) // 16)):
            table[b, pg] = next(blocks)
        k, v = (torch.randn(SINKS + kept, Hkv, D, generator=g).to(dt) for _ in range(2))
        pos = torch.tensor(list(range(SINKS)) + list(range(first, total - n)), device="cuda")
        slots = table[b, pos // 16].long() * 16 + pos % 16
        pool.append(0, k[:-n].cuda(), v[:-n].cuda(), slots)
        ks.append(k)
        vs.append(v)
        for pg in range(first // 16, (total + 15) // 16):      # hidden from every query: outside the pool again
            if pg * 16 + 16 <= total - n - WINDOW + 1:
                table[b, pg] = -1
    q = torch.randn(2, n, Hq, D, generator=g).to(dt)
    kn, vn = (torch.stack([x[-n:] for x in y]).cuda() for y in (ks, vs))
    lens = torch.tensor(totals, dtype=torch.int32, device="cuda")
    out = torch.full((2 * n, Hq, D), 7.0, dtype=dt, device="cuda")
    if n == 1:
        pool.paged_decode(0, q[:, 0].cuda(), table, lens, out, k_new=kn[:, 0].contiguous(), v_new=vn[:, 0].contiguous(),
                          window=WINDOW, sinks=SINKS)
    else:
        cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
        pool.paged_prefill(0, q.flatten(0, 1).cuda(), cu, lens - n, table, out, k_new=kn.flatten(0, 1), v_new=vn.flatten(0, 1),
                           window=WINDOW, sinks=SINKS)
    assert pool.check() == 0
    for b, total in enumerate(totals):
        # the sinks and the tail as one short sequence: a window that ends before the sinks sees them through `sinks`
        S = SINKS + kept
        ref = attend(q[b], held(ks[b], kv), held(vs[b], kv), torch.arange(S - n, S), WINDOW, SINKS, v_scale=v_scales(vs[b], kv))
        check(out[b * n:(b + 1) * n], *ref, io, kv, f"sequence {b}")
