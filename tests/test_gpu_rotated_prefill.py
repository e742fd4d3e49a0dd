"""RoPE in the prefills of 4-bit pools and under windows, and FP8's default codec under a window.

A rotated call equals the plain call over rows that the library rotated, bit for bit: outputs and pages.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import oracle  # noqa: E402
from tests.paged_cases import Batch, attend, check, held, v_scales  # noqa: E402
from tests.test_gpu_window import device_rope  # noqa: E402

pytestmark = pytest.mark.gpu

KINDS = [("fp4", "bf16", 128, 28, 4, 0, 0), ("fp4", "bf16", 64, 14, 2, 50, 3), ("fp4", "f16", 128, 16, 1, 0, 0),
         ("fp4", "f16", 64, 6, 6, 9, 1), ("bf16", "bf16", 128, 28, 4, 50, 3), ("bf16", "bf16", 64, 6, 6, 100, 0),
         ("f16", "f16", 128, 8, 2, 33, 17), ("f16", "f16", 64, 14, 2, 10, 1), ("fp8", "bf16", 128, 32, 8, 40, 4),
         ("fp8", "f16", 128, 8, 1, 40, 0)]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("chunks", [[(0, 40), (37, 1), (300, 65)], [(1500, 9)]], ids=["3", "split"])
@pytest.mark.parametrize("theta", [1e4, 1e6])
@pytest.mark.parametrize("kv,io,D,Hq,Hkv,window,sinks", KINDS)
def test_rotates_queries_and_the_chunk(kv, io, D, Hq, Hkv, window, sinks, theta, chunks):
    totals = [a + n for a, n in chunks]
    a, b = (Batch(len(chunks) + D, kv, io, D, Hq, Hkv, totals).fill([c for c, _ in chunks]) for _ in range(2))
    q = a.rows(sum(n for _, n in chunks), Hq).to(a.dev)
    cu = torch.tensor([0] + [n for _, n in chunks]).cumsum(0).int().to(a.dev)
    start = torch.tensor([c for c, _ in chunks], dtype=torch.int32, device=a.dev)
    kn = torch.cat([x[c:] for x, (c, _) in zip(a.k, chunks)]).to(a.dev)
    vn = torch.cat([x[c:] for x, (c, _) in zip(a.v, chunks)]).to(a.dev)
    at = [p + 1 for c, n in chunks for p in range(c, c + n)]
    qr, kr = device_rope(q, at, theta), device_rope(kn, at, theta)
    assert not torch.equal(qr, q) and not torch.equal(kr, kn)
    oa, ob = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    win = dict(window=window, sinks=sinks)
    a.pool.paged_prefill(0, q, cu, start, a.device_table(), oa, k_new=kn, v_new=vn, rope_theta=theta, **win)
    b.pool.paged_prefill(0, qr, cu, start, b.device_table(), ob, k_new=kr, v_new=vn, **win)
    assert a.pool.check() == b.pool.check() == 0
    assert torch.equal(a.pool.pages_u8(), b.pool.pages_u8())
    if kv == "fp8":
        assert torch.equal(a.pool.scales_f32().view(torch.int32), b.pool.scales_f32().view(torch.int32))
    assert torch.equal(oa, ob)
    for s, (c, n) in enumerate(chunks):
        rows = slice(int(cu[s]), int(cu[s + 1]))
        k = torch.cat([b.k[s][:c], kr[rows].cpu()])
        ref = attend(qr[rows].cpu(), held(k, kv), held(b.v[s], kv), torch.arange(c, c + n), window, sinks,
                     v_scale=v_scales(b.v[s], kv))
        check(oa[rows], *ref, io, kv, f"chunk {s}")


@pytest.mark.parametrize("window,sinks", [(1, 0), (17, 3), (100, 4), (2 ** 32 - 1, 0)])
@pytest.mark.parametrize("io,Hq,Hkv", [("bf16", 32, 8), ("f16", 16, 1)])
def test_fp8_default_codec_under_a_window(io, Hq, Hkv, window, sinks):
    """The truncating encoder (its largest code stands for 480): decode and prefill over the values that the pool holds."""
    chunks = [(0, 5), (700, 130), (31, 1)]
    totals = [a + n for a, n in chunks]
    bt = Batch(window % 89, "fp8", io, 128, Hq, Hkv, totals, fp8_mode="reference").fill()
    values = torch.from_numpy(oracle.fp8_decode(np.arange(256, dtype=np.uint8))).double()
    k, v, t = [], [], []
    for b, n in enumerate(totals):
        ck, cv, ks, vs = bt.pool.gather(0, bt.device_table()[b], n)
        k.append((values[ck.cpu().long()] * ks.cpu().double()[..., None]).transpose(0, 1))
        v.append((values[cv.cpu().long()] * vs.cpu().double()[..., None]).transpose(0, 1))
        t.append(vs.cpu().double().transpose(0, 1))
    q = [bt.rows(n, Hq) for _, n in chunks]
    qd, last = torch.cat(q).to(bt.dev), torch.stack([x[-1] for x in q]).to(bt.dev)
    cu = torch.tensor([0] + [n for _, n in chunks]).cumsum(0).int().to(bt.dev)
    start = torch.tensor([a for a, _ in chunks], dtype=torch.int32, device=bt.dev)
    out, dec = torch.full_like(qd, 7.0), torch.full_like(last, 7.0)
    bt.pool.paged_prefill(0, qd, cu, start, bt.device_table(), out, window=window, sinks=sinks)
    bt.pool.paged_decode(0, last, bt.device_table(), bt.lens(), dec, window=window, sinks=sinks)
    assert bt.pool.check() == 0
    for b, (a, n) in enumerate(chunks):
        ref = attend(q[b], k[b], v[b], torch.arange(a, a + n), window, sinks, v_scale=t[b])
        check(out[int(cu[b]):int(cu[b + 1])], *ref, io, "fp8", f"chunk {b}")
        check(dec[b:b + 1], *(x[-1:] for x in ref), io, "fp8", f"decode {b}")
