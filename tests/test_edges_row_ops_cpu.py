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


# ---------------------------------------------------------------------------------------------------------------- AdamW's checkpoints
@pytest.fixture
def AdamW(hip, monkeypatch):
    """The optimizer with its host code alone: parameters on the CPU, no step."""
    from virconv_amd import optim
    monkeypatch.setattr(optim.AdamW, "_check_group", lambda self, g: None)
    return optim.AdamW


def moments(opt, p, seed):
    """Random 8-bit moments, over a few binades, some zero, one undefined."""
    g = torch.Generator().manual_seed(seed)
    st = opt._new_state(p)
    n, blocks = p.numel(), -(-p.numel() // 128)
    for k in ("exp_avg", "exp_avg_rms"):
        v = torch.randn(n, generator=g) * torch.exp(2 * torch.randn(n, generator=g))
        v = (v.abs() if k == "exp_avg_rms" else v).clamp(-250, 250) * (torch.rand(n, generator=g) > 0.1)
        v[0] = float("nan")
        torch.as_strided(st[k].view(torch.uint8), (n,), (1,)).copy_(v.to(torch.float8_e4m3fn).view(torch.uint8))
    st["exponents"].copy_(torch.randint(-20, 3, (blocks, 2), generator=g))
    st["step"] = 7
    return st


@pytest.mark.parametrize("shape", [(8, 16, 3, 3), (5, 7, 2, 3), (130, 3, 1, 2)], ids=str)
@pytest.mark.parametrize("back", [False, True])
def test_8_bit_moments_survive_a_change_of_memory_order(AdamW, shape, back):
    g = torch.Generator().manual_seed(1)
    p = torch.nn.Parameter(torch.randn(shape, generator=g))
    q = torch.nn.Parameter(p.detach().to(memory_format=torch.channels_last))
    p, q = (q, p) if back else (p, q)
    one, two = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
    moments(one, p, 2)
    two.load_state_dict(one.state_dict())
    want, got = one.decoded_state(p), two.decoded_state(q)
    assert two.state[q]["step"] == 7 and all(t.stride() == q.stride() for t in got)
    st = two.state[q]
    for k, column, (a, b) in (("exp_avg", 0, (want[0], got[0])), ("exp_avg_rms", 1, (want[1].sqrt(), got[1].sqrt()))):
        unit = torch.empty_like(q, dtype=torch.float64)
        torch.as_strided(unit, (q.numel(),), (1,)).copy_((2.0 ** (st["exponents"][:, column].double() - 7)).repeat_interleave(128, 0)[:q.numel()])
        nan = torch.isnan(a)
        assert torch.equal(torch.isnan(b), nan) and int(nan.sum()) == 1
        # to the nearest e4m3 value: 2^-4 of it, or half of the smallest ones' distance 2^-9; a root up to all of that (and the squares' own rounding)
        bound = torch.maximum((2.0 ** -4 + 1e-6) * a.double().abs(), unit * 2.0 ** (-10 if column == 0 else -9))
        assert bool(((a.double() - b.double()).abs() <= bound)[~nan].all())
        assert bool((b[~nan & (a != 0)] != 0).all()) or column == 0


@pytest.mark.parametrize("like", ["equal", "axes of one element"])
def test_8_bit_moments_of_the_same_memory_order_stay_bit_for_bit(AdamW, like):
    shape = (40, 1, 5, 6) if like != "equal" else (8, 16, 3, 3)
    p = torch.nn.Parameter(torch.randn(shape))
    q = torch.nn.Parameter(torch.empty_strided(shape, (30, 1, 6, 1)).copy_(p.detach()) if like != "equal" else p.detach().clone())
    one, two = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
    a = moments(one, p, 3)
    two.load_state_dict(one.state_dict())
    b = two.state[q]
    assert torch.equal(a["exponents"], b["exponents"])
    assert all(torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)) for k in ("exp_avg", "exp_avg_rms"))


def test_a_moment_whose_blocks_are_not_known_is_refused(AdamW):
    p = torch.nn.Parameter(torch.randn(16, 24))
    opt = AdamW([p], state_bits=8)
    moments(opt, p, 4)
    saved = opt.state_dict()
    saved["state"][0]["exp_avg"] = torch.zeros(16, 48, dtype=torch.uint8)[:, ::2].view(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="not dense"):
        AdamW([p], state_bits=8).load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_of_steps_that_are_not_done_here_are_refused(AdamW, bits):
    p = torch.nn.Parameter(torch.randn(16, 24))
    p.grad = torch.randn(16, 24)
    before = p.detach().clone()

    def saved(kind, **options):
        q = torch.nn.Parameter(p.detach().clone())
        q.grad = p.grad.clone()
        opt = kind([q], lr=1e-3, weight_decay=0.01, **options)
        opt.step()
        return opt.state_dict()

    ours = AdamW([p], lr=2e-3, state_bits=bits)
    for state, word in ((saved(torch.optim.AdamW, maximize=True), "maximize"), (saved(torch.optim.AdamW, amsgrad=True), "amsgrad"),
                        (saved(torch.optim.Adam), "adds its weight decay")):
        with pytest.raises(ValueError, match=word):
            ours.load_state_dict(state)
        assert ours.param_groups[0]["lr"] == 2e-3 and p not in ours.state and torch.equal(p, before)       # nothing of it was taken
    if bits == 32:
        ours.load_state_dict(saved(torch.optim.AdamW))
        assert ours.state[p]["step"] == 1 and ours.param_groups[0]["lr"] == 1e-3
        with pytest.raises(ValueError, match="state_bits"):
            other = AdamW([p], state_bits=8)
            moments(other, p, 1)
            AdamW([p]).load_state_dict(other.state_dict())


def test_8_bit_states_that_lack_a_moment_are_refused(AdamW):
    p = torch.nn.Parameter(torch.randn(16, 24))
    opt = AdamW([p], state_bits=8)
    moments(opt, p, 5)
    saved = opt.state_dict()
    del saved["state"][0]["exp_avg_rms"]
    with pytest.raises(ValueError, match="without 'exp_avg_rms'"):
        AdamW([p], state_bits=8).load_state_dict(saved)


# ---------------------------------------------------------------------------------------------------------------- the native host side
@pytest.mark.parametrize("what", ["missing", "of another layout", "of another torch", "no extension"])
def test_what_does_not_use_the_native_host_side_does_without_it(what, monkeypatch, tmp_path):
    from virconv_amd.backend_hip import HipBackend
    monkeypatch.setattr(_lib, "_host", None)
    if what == "missing":
        monkeypatch.setattr(_lib, "HOST_PATH", str(tmp_path / "_host_ops.so"))
    elif what == "no extension":
        (tmp_path / "_host_ops.so").write_bytes(b"no shared object")
        monkeypatch.setattr(_lib, "HOST_PATH", str(tmp_path / "_host_ops.so"))
    elif what == "of another torch":
        monkeypatch.setattr(torch, "__version__", "0.0")
    else:
        monkeypatch.setattr(_lib, "ABI_VERSION", _lib.ABI_VERSION + 1)
    with ops.use_backend(HipBackend()) as be:     # everything that goes through the C ABI alone
        assert be.lib.vc_abi_version() > 0
        with pytest.raises(_lib.VirConvError, match="python -m virconv_amd.build"):
            ops.layer_norm(torch.zeros(2, 4))
        with pytest.raises(_lib.VirConvError, match="python -m virconv_amd.build"):
            be.host
    monkeypatch.undo()
    assert _lib.load_host().ABI_VERSION == _lib.ABI_VERSION


# ---------------------------------------------------------------------------------------------------------------- derivatives
@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(hip, which):
    """(They are refused before a tensor's device is looked at.)"""
    from torch.autograd import forward_ad
    norm = [torch.randn(4, 8), torch.randn(8), torch.randn(8)]
    grouped = [torch.randn(4, 8), torch.randn(2, 5, 8), torch.randn(2, 5)]
    offsets = torch.tensor([0, 1, 4])
    with forward_ad.dual_level():
        for args in (norm, grouped):
            args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="layer_norm: no forward-mode"):
            ops.layer_norm(*norm)
        with pytest.raises(NotImplementedError, match="grouped_linear: no forward-mode"):
            ops.grouped_linear(grouped[0], grouped[1], offsets, grouped[2])
    with pytest.raises(_lib.VirConvError, match="no CPU path"):
        ops.layer_norm(torch.randn(4, 8))


# ---------------------------------------------------------------------------------------------------------------- AdamW's states
def test_a_state_handed_to_another_parameter_is_followed(AdamW):
    a, b, c = (torch.nn.Parameter(torch.zeros(4)) for _ in range(3))
    opt = AdamW([a, b, c])
    group = opt.param_groups[0]["params"]
    one, two = opt._new_state(a), opt._new_state(c)
    same = lambda *want: all(x is y for x, y in zip(opt._states_of(0, group), want))     # noqa: E731
    assert same(one, None, two) and same(one, None, two)
    opt.state[b] = opt.state.pop(c)                    # the same dicts in the same order, one of them for another parameter
    assert same(one, two, None)
    opt.state[a], opt.state[b] = opt.state[b], opt.state[a]
    assert same(two, one, None)
    group[0], group[1] = b, a
    assert same(one, two, None)
    del opt.state[a]
    assert same(one, None, None)


def test_a_first_group_without_parameters(hip):
    from virconv_amd.optim import AdamW
    with pytest.raises(ValueError, match="no CPU path"):       # (of the second group's parameter)
        AdamW([{"params": []}, {"params": [torch.nn.Parameter(torch.zeros(4))]}])


def test_capture_is_looked_for_on_the_device_of_the_parameters(AdamW, monkeypatch):
    """The first step, parameters of other memory orders: the path in Python.  (The current stream is one of the current device.)"""
    inside = []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            inside.append(self.device)

        def __exit__(self, *error):
            inside.pop()

    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: inside == [p.device])
    with pytest.raises(RuntimeError, match="captured"):
        AdamW([p]).step()


# ---------------------------------------------------------------------------------------------------------------- sizes
def test_layer_norm_refuses_what_one_launch_cannot_hold():
    fake = ctypes.c_void_p(4096)    # never dereferenced on the host
    f, b = _lib.load().vc_layer_norm_forward, _lib.load().vc_layer_norm_backward

    def refused(status):
        return status == _lib.VC_EINVAL and b"too many for one launch" in _lib.load().vc_last_error()

    for c, dtype in ((16385, 0), (16385, 2), (1 << 20, 1)):
        assert refused(f(fake, c, 1 << 22, c, dtype, None, 0, None, 0, 1e-5, fake, None, None, None))
        assert refused(b(fake, c, fake, c, 1 << 22, c, dtype, None, 0, 0, fake, fake, fake, None, None, None, 0, None))
    for dw, db in ((fake, None), (None, fake)):
        assert refused(b(fake, 1 << 27, fake, 1 << 27, 1, 1 << 27, 0, None, 0, 0, fake, fake, None, dw, db, fake, 1 << 40, None))
