"""The 4-bit pool's refusals and sizes on the CPU, and the reference codec of its tests against its definition."""
import ctypes
import math

import pytest

from voidweb_b200 import _lib as C

torch = pytest.importorskip("torch")
from tests.paged_cases import held  # noqa: E402


def create(D=128, kv=C.VW_FP4_E2M1, io=C.VW_BF16, blocks=8, data=None):
    cfg = C.PoolConfig(1, 2, D, blocks, kv, io, 0, 8, 0, 0, data, None)
    h = ctypes.c_void_p()
    return C.lib().vw_pool_create(ctypes.byref(cfg), ctypes.byref(h))


def test_pool_refusals():
    assert create(D=96) == C.VW_ERR_UNSUPPORTED
    assert create(D=32) == C.VW_ERR_UNSUPPORTED
    assert create(kv=4) == C.VW_ERR_INVALID_ARG
    assert create(io=C.VW_FP4_E2M1) == C.VW_ERR_INVALID_ARG
    assert create(blocks=0) == C.VW_ERR_INVALID_ARG
    assert create(data=256 + 16) == C.VW_ERR_INVALID_ARG


def test_block_bytes():
    from voidweb_b200.kv import PoolSpec
    assert PoolSpec(28, 4, 128, 10, kv_dtype="fp4").block_bytes == 28 * 4 * 2304
    assert PoolSpec(1, 2, 64, 10, kv_dtype="fp4").block_bytes == 2 * 1152


def test_reference_codec_is_the_nearest_code():
    """held() against a search over all 16 codes and all E4M3 scales."""
    codes = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    scales = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    scales = scales[(scales >= 0) & scales.isfinite()].unique()
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(400, 16, generator=g) * 2.0 ** torch.randint(-12, 12, (400, 1), generator=g)).bfloat16()
    got = held(x, "fp4")
    for r in range(400):
        row = x[r].double()
        want = row.abs().max().item() / 6
        d = (scales - want).abs()
        near = scales[d == d.min()]
        for i in range(16):
            options = {0.0} if 0.0 in near.tolist() else set()
            for s in near[near > 0].tolist():
                far = (abs(row[i].item()) / s - codes).abs()
                options |= {c * s for c in codes[far == far.min()].tolist()}
            assert abs(got[r, i].item()) in options and got[r, i] * row[i] >= 0


def _borders_code(v):
    """E2M1 magnitude code of a quotient, to nearest, ties to even."""
    return (v > .25) * 1 + (v >= .75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5)


@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_products_decide_codes_as_quotients_do(io):
    """vw_fp4.cuh's arithmetic, restated in f32: every magnitude of the io type as a group's maximum, and every magnitude
    under every scale with an inverse one ulp off either way, against the real quotients."""
    import numpy as np
    f = np.float32
    bits = np.arange(0, 0x7F80 if io == "bf16" else 0x7C00, dtype=np.uint16)
    x = (bits.astype(np.uint32) << 16).view(f) if io == "bf16" else bits.view(np.float16).astype(f)

    def e4m3(v):
        e = np.maximum(np.floor(np.log2(np.maximum(v, 1e-300))), -6)
        step = 2.0 ** (e - 3)
        return np.minimum(np.round(v / step) * step, 448.0)

    t = np.minimum(x, f(1048576)) * f(1 / 6)
    c = t * f(513)
    want = e4m3(np.minimum(x.astype(np.float64) / 6, 448))
    assert (e4m3((c - (c - t)).astype(np.float64)) == want).all()
    xs = x[(x > 0) & (x < 1e6)]
    for s in np.unique(want[want > 0]):
        real = _borders_code(xs.astype(np.float64) / s)
        inv = f(1 / s)
        for r in (inv, np.nextafter(inv, f(0)), np.nextafter(inv, f(np.inf))):
            q = (xs * r + f(1536)) - f(1536)
            assert (_borders_code(q.astype(np.float64)) == real).all(), s


def test_division_by_heads_as_a_product():
    """vw_kv_ops.cu's HeadDiv over row counts below 2^31."""
    import random
    rng = random.Random(1)
    for d in list(range(1, 130)) + [1000, 65535]:
        s = 0
        while (1 << s) < d:
            s += 1
        m = ((1 << (31 + s)) + d - 1) // d
        assert m < 1 << 32
        for w in list(range(300)) + [2 ** 31 - 1 - i for i in range(300)] + [rng.randrange(2 ** 31) for _ in range(300)]:
            assert w * m >> (31 + s) == w // d
