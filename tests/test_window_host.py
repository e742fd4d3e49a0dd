"""Windowed calls on the CPU: refusals that need no pool, and the pages that a window visits."""
import ctypes

import pytest

from voidweb_b200 import _lib as C


def test_null_arguments_are_refused():
    L = C.lib()
    w = C.Window(4, 0)
    assert L.vw_paged_decode_window(None, None, ctypes.byref(w), None) == C.VW_ERR_INVALID_ARG
    assert L.vw_paged_prefill_window(None, None, ctypes.byref(w), None) == C.VW_ERR_INVALID_ARG
    assert L.vw_decode_step_host_window(None, None, ctypes.byref(w), None) == C.VW_ERR_INVALID_ARG
    assert L.vw_decode_step_host_window(None, None, None, None) == C.VW_ERR_INVALID_ARG
    assert b"window" in L.vw_last_error()
    assert L.vw_decode_step_host_window(None, None, ctypes.byref(C.Window(0, 3)), None) == C.VW_ERR_INVALID_ARG


def test_injected_faults_reach_the_windowed_calls():
    L = C.lib()
    w = C.Window(4, 0)
    for f in (L.vw_paged_decode_window, L.vw_paged_prefill_window, L.vw_decode_step_host_window):
        assert L.vw_fault_inject(C.VW_FAULT_CUDA, 1) == C.VW_OK
        assert f(None, None, ctypes.byref(w), None) == C.VW_ERR_CUDA
        assert L.vw_fault_pending(C.VW_FAULT_CUDA) == 0


def test_python_window_arguments():
    torch = pytest.importorskip("torch")
    assert torch is not None
    from voidweb_b200.kv import _window
    assert _window(0, 0) is None
    w = _window(2 ** 32 - 1, 7)
    assert (w.window, w.sinks) == (2 ** 32 - 1, 7)
    for bad in ((0, 1), (-1, 0), (1, -1), (2 ** 32, 0), (1, 2 ** 32)):
        with pytest.raises(ValueError):
            _window(*bad)


def span(np_, first, window, sinks):
    """vw_window.cuh's page_span, restated."""
    lo = max(0, first + 1 - window)
    ns = (min(sinks, lo) + 15) // 16
    skip = max(0, lo // 16 - ns)
    return np_ - skip, ns, skip, lo


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 33, 100, 1 << 30])
@pytest.mark.parametrize("sinks", [0, 1, 15, 16, 17, 40, 1 << 30])
def test_visited_pages_are_those_with_a_visible_token(window, sinks):
    for total in (1, 2, 15, 16, 17, 32, 33, 48, 100, 130):
        for first in range(max(0, total - 40), total):          # queries first .. total - 1
            np_ = (total + 15) // 16
            n, ns, skip, lo = span(np_, first, window, sinks)
            pages = [o if o < ns else o + skip for o in range(n)]
            seen = sorted({j // 16 for p in range(first, total) for j in range(p + 1) if p - j < window or j < sinks})
            assert pages == seen
            for pg in pages:
                a, b = max(0, sinks - pg * 16), min(16, lo - pg * 16)
                for r in range(16):
                    j = pg * 16 + r
                    anyone = any(p - j < window or j < sinks for p in range(first, total) if p >= j)
                    if j < total:
                        assert (not (a <= r < b)) == anyone
