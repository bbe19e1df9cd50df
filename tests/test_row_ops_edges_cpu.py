"""Layer norm, grouped products and the optimizers where a user's program meets something unusual: what can be checked without a GPU."""
import ctypes

import pytest
import torch

from virconv_amd import _lib, ops


@pytest.fixture
def hip():
    from virconv_amd.backend_hip import HipBackend
    with ops.use_backend(HipBackend()) as be:
        yield be


# ---------------------------------------------------------------------------------------------------------------- AdamW's tensors in memory
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("count", [2, 5, 140])
def test_overlaps_of_any_two_written_tensors_are_refused(count, order, bits):
    f = _lib.load().vc_adamw
    n, kinds = 256, 4 if bits == 8 else 3
    places = list(range(count))
    if order == "falling":
        places.reverse()
    if order == "mixed":
        places = [(7 * k + 3) % count for k in range(count)] if count % 7 else [places[k // 2] if k % 2 else places[-1 - k // 2] for k in range(count)]
    assert sorted(places) == list(range(count))
    size = {0: 4 * n, 1: n * bits // 8, 2: n * bits // 8, 3: 2 * n // 128}
    base = lambda kind, k: (1 + kind) << 32 | places[k] * 4096        # noqa: E731

    def refused(moved, onto):
        """Is a step refused whose tensor `moved` (kind, index) begins in the last bytes of `onto`?"""
        t = (ctypes.c_int64 * (7 * count))()
        for k in range(count):
            row = {kind: base(kind, k) for kind in range(4)}
            if moved[1] == k:
                unit = {0: 4, 3: 1}.get(moved[0], bits // 8)
                row[moved[0]] = base(*onto) + size[onto[0]] - unit
            t[7 * k: 7 * k + 7] = [row[0], 1 << 40, row[1], row[2], row[3], n, k]
        status = f(ctypes.cast(t, ctypes.c_void_p), count, 0, bits, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, 0, None)
        return status == _lib.VC_EINVAL and b"overlap" in _lib.load().vc_last_error()

    for a in range(kinds):
        for b in range(kinds):
            for i, j in ((0, count - 1), (count - 1, 0), (count // 2, 0)):
                if (a, i) != (b, j):
                    assert refused((a, i), (b, j)), (a, i, b, j)
