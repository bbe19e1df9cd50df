"""Layer norm, grouped products and the multi-tensor AdamW step: what is refused, and refused before anything reaches a GPU; the module
layouts; the 8-bit state's arithmetic against its definition."""
import ctypes

import pytest
import torch

from virconv_amd import _lib, ops
from virconv_amd.row_layers import GroupedLinear, LayerNorm
from rowref import decode_blocks, encode_blocks, mix32

FAKE = ctypes.c_void_p(4096)    # never dereferenced on the host


@pytest.fixture
def hip():
    from virconv_amd.backend_hip import HipBackend
    with ops.use_backend(HipBackend()) as be:
        yield be


def refused(status, text):
    assert status == _lib.VC_EINVAL
    assert text in _lib.load().vc_last_error(), _lib.load().vc_last_error()


def test_layer_norm_abi_refusals():
    f, b = _lib.load().vc_layer_norm_forward, _lib.load().vc_layer_norm_backward
    refused(f(FAKE, 8, 4, 8, 3, None, 0, None, 0, 1e-5, FAKE, None, None, None), b"dtype")
    refused(f(FAKE, 8, 4, 8, 0, None, 5, None, 0, 1e-5, FAKE, None, None, None), b"dtype")
    refused(f(FAKE, 8, -1, 8, 0, None, 0, None, 0, 1e-5, FAKE, None, None, None), b"rows")
    refused(f(FAKE, 8, 4, 0, 0, None, 0, None, 0, 1e-5, FAKE, None, None, None), b"rows")
    refused(f(FAKE, 7, 4, 8, 0, None, 0, None, 0, 1e-5, FAKE, None, None, None), b"stride")
    refused(f(FAKE, 8, 4, 8, 0, None, 0, None, 0, 1e-5, FAKE, FAKE, None, None), b"come together")
    refused(f(None, 8, 4, 8, 0, None, 0, None, 0, 1e-5, FAKE, None, None, None), b"NULL")
    assert f(None, 8, 0, 8, 0, None, 0, None, 0, 1e-5, None, None, None, None) == _lib.VC_OK
    refused(b(FAKE, 8, FAKE, 7, 4, 8, 0, None, 0, 0, FAKE, FAKE, FAKE, None, None, None, 0, None), b"stride")
    refused(b(FAKE, 8, FAKE, 8, 4, 8, 0, None, 0, 0, None, FAKE, FAKE, None, None, None, 0, None), b"NULL")
    need = _lib.load().vc_layer_norm_backward_workspace_bytes(4, 8, 0)
    assert need > 0 and _lib.load().vc_layer_norm_backward_workspace_bytes(0, 8, 0) == 0
    refused(b(FAKE, 8, FAKE, 8, 4, 8, 0, None, 0, 0, FAKE, FAKE, None, FAKE, None, FAKE, need - 1, None), b"workspace")
    refused(b(FAKE, 8, FAKE, 8, 4, 8, 0, None, 0, 0, FAKE, FAKE, None, None, FAKE, None, need, None), b"workspace")


def test_grouped_linear_abi_refusals():
    lib = _lib.load()
    f, i, w, size = (lib.vc_grouped_linear_forward, lib.vc_grouped_linear_backward_input, lib.vc_grouped_linear_backward_weight,
                     lib.vc_grouped_linear_workspace_bytes)
    refused(f(FAKE, 8, 4, FAKE, None, FAKE, 16, 2, 8, 8, 0, FAKE, None, 0, None), b"offsets of 16 bits")
    refused(f(FAKE, 8, 4, FAKE, None, FAKE, 32, 2, 8, 8, 4, FAKE, None, 0, None), b"dtype")
    refused(f(FAKE, 8, 1 << 31, FAKE, None, FAKE, 32, 2, 8, 8, 0, FAKE, None, 0, None), b"rows")
    refused(f(FAKE, 8, 4, FAKE, None, FAKE, 32, 2, 0, 8, 0, FAKE, None, 0, None), b"channels")
    refused(f(FAKE, 8, 4, FAKE, None, None, 32, 2, 8, 8, 0, FAKE, None, 0, None), b"offsets")
    refused(f(FAKE, 7, 4, FAKE, None, FAKE, 32, 2, 8, 8, 0, FAKE, None, 0, None), b"stride")
    refused(f(FAKE, 8, 4, None, None, FAKE, 32, 2, 8, 8, 0, FAKE, None, 0, None), b"NULL")
    refused(i(FAKE, 7, 4, FAKE, FAKE, 32, 2, 8, 8, 0, FAKE, None, 0, None), b"stride")
    refused(w(FAKE, 8, FAKE, 7, 4, FAKE, 32, 2, 8, 8, 0, FAKE, None, None, 0, None), b"stride")
    refused(w(FAKE, 8, None, 8, 4, FAKE, 32, 2, 8, 8, 0, FAKE, None, None, 0, None), b"NULL")
    # a long inner axis with few rows is split, and its partial sums need room
    need = size(0, 480, 3, 27648, 256, 0)
    assert need >= 2 * 480 * 256 * 4
    refused(f(FAKE, 27648, 480, FAKE, None, FAKE, 32, 3, 27648, 256, 0, FAKE, FAKE, need - 1, None), b"workspace")
    need = size(2, 133578, 4, 64, 64, 0)
    assert need >= 4 * 64 * 64 * 4
    refused(w(FAKE, 64, FAKE, 64, 133578, FAKE, 32, 4, 64, 64, 0, FAKE, None, None, need, None), b"workspace")
    assert size(0, 0, 3, 8, 8, 0) == 0 and size(0, 8, 0, 8, 8, 0) == 0
    assert f(None, 8, 0, None, None, FAKE, 32, 2, 8, 8, 0, None, None, 0, None) == _lib.VC_OK
    assert w(None, 8, None, 8, 0, None, 32, 0, 8, 8, 0, None, None, None, 0, None) == _lib.VC_OK


def table(*rows):
    t = (ctypes.c_int64 * (7 * len(rows)))()
    for k, r in enumerate(rows):
        for j, v in enumerate(r):
            t[7 * k + j] = v
    return ctypes.cast(t, ctypes.c_void_p)


def test_adamw_abi_refusals():
    f = _lib.load().vc_adamw
    ok = (0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 16, 0)
    go = lambda t, n=1, dtype=0, bits=32, b1=0.9, b2=0.99, step=1: f(t, n, dtype, bits, 1e-3, b1, b2, 1e-8, 0.01, step, 0, None)  # noqa: E731
    refused(go(table(ok), dtype=3), b"dtype")
    refused(go(table(ok), bits=16), b"16 bits")
    refused(go(table(ok), step=0), b"first step")
    refused(go(table(ok), b1=1.0), b"betas")
    refused(go(None), b"tensors")
    refused(go(table((0x1000, 0, 0x3000, 0x4000, 0, 16, 0))), b"NULL")
    refused(go(table((0x1000, 0x2000, 0x3000, 0x4000, 0, 16, 0)), bits=8), b"NULL")
    refused(go(table((0x1002, 0x2000, 0x3000, 0x4000, 0, 16, 0))), b"aligned")
    refused(go(table((0x1000, 0x2000, 0x3000, 0x4000, 0, -1, 0))), b"n = -1")
    refused(go(table((0x1000, 0x2000, 0x3000, 0x4000, 0, 16, 1 << 20))), b"place")
    refused(go(table((0x1000, 0x2000, 0x3000, 0x3020, 0, 16, 0))), b"overlap")
    refused(go(table(ok, (0x103c, 0x2000, 0x6000, 0x7000, 0, 16, 0)), n=2), b"overlap")
    assert go(table((0, 0, 0, 0, 0, 0, 0))) == _lib.VC_OK and go(None, n=0) == _lib.VC_OK


def test_python_refusals(hip):
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(_lib.VirConvError, match="no CPU path"):
        ops.layer_norm(x, w)
    with pytest.raises(ValueError, match="weight has shape"):
        ops.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="bias is"):
        ops.layer_norm(x, w, torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="at least one channel"):
        ops.layer_norm(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(x, w, eps=float("nan"))
    with pytest.raises(_lib.VirConvError, match="float32, float16 or bfloat16"):
        ops.layer_norm(x.double())
    weight, offsets = torch.zeros(2, 5, 8), torch.tensor([0, 1, 4])
    with pytest.raises(_lib.VirConvError, match="no CPU path"):
        ops.grouped_linear(x, weight, offsets)
    for bad in (torch.zeros(2, 5, 7), torch.zeros(5, 8), torch.zeros(2, 0, 8)):
        with pytest.raises(ValueError, match="wants x"):
            ops.grouped_linear(x, bad, offsets)
    with pytest.raises(ValueError, match="one type"):
        ops.grouped_linear(x, weight.half(), offsets)
    for bad in (offsets[:2], offsets.float(), offsets[None]):
        with pytest.raises(ValueError, match="offsets"):
            ops.grouped_linear(x, weight, bad)
    with pytest.raises(ValueError, match="bias has shape"):
        ops.grouped_linear(x, weight, offsets, torch.zeros(5))
    with pytest.raises(ValueError, match="last axis"):
        LayerNorm((4, 8))
    with pytest.raises(ValueError, match="channels"):
        LayerNorm(8)(torch.zeros(4, 7))
    with pytest.raises(ValueError, match="groups"):
        GroupedLinear(0, 8, 8)


def test_adamw_python_refusals(hip):
    from virconv_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="16 bits"):
        AdamW([p], state_bits=16)
    with pytest.raises(ValueError, match="no CPU path"):
        AdamW([p])


def test_modules_have_the_stock_layout():
    ours, stock = LayerNorm(16), torch.nn.LayerNorm(16)
    assert {k: v.shape for k, v in ours.state_dict().items()} == {k: v.shape for k, v in stock.state_dict().items()}
    m = GroupedLinear(3, 16, 8)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {"weight": (3, 8, 16), "bias": (3, 8)}
    assert float(m.weight.abs().max()) <= 0.25 and "bias=False" in repr(GroupedLinear(3, 16, 8, bias=False))
    assert list(LayerNorm(16, bias=False).state_dict()) == ["weight"] and not LayerNorm(16, elementwise_affine=False).state_dict()


# ------------------------------------------------------------------ the 8-bit state's definition (rowref), which the GPU test is held to
def test_eight_bit_values_are_neighbours_and_unbiased():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(128, generator=g) * torch.exp(3 * torch.randn(128, generator=g))
    n = 4000
    bits = torch.randint(0, 1 << 16, (n, 128), generator=g)
    codes, e = encode_blocks(x.expand(n, 128).contiguous(), bits)
    got = decode_blocks(codes, e).double()
    unit = 2.0 ** (float(torch.floor(torch.log2(x.abs().max()))) - 7)
    y = x.double().abs() / unit
    step = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3) * unit       # the grid around each value
    assert bool(((got - x.double()).abs() < step * (1 + 1e-6)).all())
    # the mean of n draws of a value that is `step` apart with probability q: sd = step sqrt(q (1 - q) / n) <= step / (2 sqrt(n)); five of
    # them, and the 2^-16 granularity of the draw
    assert bool(((got.mean(0) - x.double()).abs() <= step * (5 * 0.5 / n ** 0.5 + 2.0 ** -16)).all())


def test_eight_bit_values_on_the_grid_stay():
    e4m3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    e4m3 = e4m3[torch.isfinite(e4m3) & (e4m3.abs() < 256)]
    x = torch.cat([e4m3, torch.full((256 - e4m3.numel(),), 128.0)]).view(2, 128) * 2.0 ** -30
    x[:, 0] = 128.0 * 2.0 ** -30      # both blocks' largest magnitudes lie in the top binade
    codes, e = encode_blocks(x, torch.full((2, 128), 65535))
    assert torch.equal(decode_blocks(codes, e), x)


def test_mixing_function_is_a_permutation_with_known_values():
    # MurmurHash3's finalizer: fmix32(0) = 0, fmix32(1) = 0x514e28b7
    assert mix32(0) == 0 and mix32(1) == 0x514E28B7
    x = torch.arange(1 << 16)
    assert torch.unique(mix32(x)).numel() == 1 << 16
