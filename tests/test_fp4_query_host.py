"""The powers of two that bring bf16 query rows into f16 over 4-bit pools, restated: every largest element a row can have."""
import pytest

torch = pytest.importorskip("torch")


def factor(top):
    """vw_fp4.cuh's fp4_query_factor."""
    e = (top >> 7) - 127
    if top == 0 or e == 128 or -1 <= e < 16:
        return 1.0
    return 2.0 ** min(14 - e, 126)


def test_every_row_fits_f16():
    bits = torch.arange(1, 0x7F80, dtype=torch.int32)
    tops = (bits << 16).view(torch.float32).double()
    for top, v in zip(bits.tolist()[::7], tops.tolist()[::7]):
        f = factor(top)
        assert 0.0 < v * f < 65504.0
        assert f == 1.0 or f >= 2.0 ** -126 and 1.0 / f >= 2.0 ** -126     # both normal in 32 bits
        # an element of the row keeps its value to 2^-24 of the row's largest
        for x in (v, v * 2.0 ** -9, v * 2.0 ** -20 * 1.0078125):
            x = torch.tensor(x).bfloat16().double()
            kept = (x * f).half().double() / f
            assert abs(kept - x) <= v * 2.0 ** -24
    assert all(factor(t) == 1.0 for t in (0, 0x7F80, 0x7FC0, 0x3F00, 0x477F))
