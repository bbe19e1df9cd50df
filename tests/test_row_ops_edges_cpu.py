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


# ---------------------------------------------------------------------------------------------------------------- fp32 operands in three pieces
def pieces(x):
    """x = h + m + l as the kernels form them: each rounded to nearest bf16."""
    h = x.bfloat16().float()
    m = (x - h).bfloat16().float()
    return h, m, (x - h - m).bfloat16().float()


def test_pieces_are_exact_and_what_is_left_out_of_a_product_is_below_two_to_the_minus_24():
    # every mantissa: the sizes of the pieces, relative to the value, and that nothing is left
    x = (torch.arange(1 << 23, dtype=torch.int32) | 127 << 23).view(torch.float32)
    h, m, low = (t.double() for t in pieces(x))
    assert torch.equal(h + m + low, x.double())
    m, low = m.abs() / x.double(), low.abs() / x.double()
    assert float(m.max()) <= 2.0 ** -8 and float(low.max()) <= 2.0 ** -17
    # m_x l_y + l_x m_y + l_x l_y over the worst pairs: those among the mantissas with the largest m, the largest l and the largest products of both
    worst = torch.cat([t.topk(300).indices for t in (m, low, m * low, m + 512 * low)] + [torch.randint(0, 1 << 23, (300,), generator=torch.Generator().manual_seed(0))])
    a, b = m[worst], low[worst]
    assert float((a[:, None] * b + b[:, None] * a + b[:, None] * b).max()) <= 2.0 ** -24
    # 1.03125 - 2^-23 squared, of which pieces that are cut off instead leave out 7.8 * 2^-24
    cut = lambda t: (t.view(torch.int32) & -65536).view(torch.float32)        # noqa: E731
    v = torch.tensor([1 + 2.0 ** -7 - 2.0 ** -23])
    for form, low_, high in ((lambda t: cut(t), 7, 8), (lambda t: t.bfloat16().float(), -1, 1)):
        h = form(v)
        m = form(v - h)
        rest = v - h - m
        h, m, rest = h.double(), m.double(), rest.double()
        kept = 2 * rest * h + m * m + 2 * m * h + h * h
        assert low_ <= float((v.double() ** 2 - kept) / v.double() ** 2 * 2.0 ** 24) <= high
