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
