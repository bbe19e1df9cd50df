"""Layer norm, grouped products and the optimizers where a user's program meets something unusual: what else holds on to the tensors that a step
writes, values that are not finite, products of worst-case mantissas, graphs with nodes in between.

Tolerances are bounds, not fits: u = 2^-24 is half a step of fp32."""
import copy
import ctypes
import math

import pytest
import torch

from rowref import floor_step, half_step

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)


def rnd(shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


# ---------------------------------------------------------------------------------------------------------------- who else sees a step
@pytest.mark.parametrize("channels_last", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_raises_the_version_of_what_it_writes(hip_backend, bits, channels_last):
    from virconv_amd.optim import AdamW
    ps = [torch.nn.Parameter(rnd((8, 6, 3, 5), 1)), torch.nn.Parameter(rnd((70,), 2, BF16)), torch.nn.Parameter(rnd((9,), 3))]
    if channels_last:     # (such a group takes the path for parameters of any order)
        ps[0] = torch.nn.Parameter(ps[0].detach().to(memory_format=torch.channels_last))
    opt = AdamW(ps, state_bits=bits, **HYPER)
    for t in range(3):
        for k, p in enumerate(ps):
            p.grad = rnd(p.shape, 10 * t + k, p.dtype) if k < 2 else None
        written = ps[:2] + [v for p in ps[:2] if p in opt.state for v in opt.state[p].values() if torch.is_tensor(v)]
        read = [ps[2], *(p.grad for p in ps[:2])]
        before = [v._version for v in written], [v._version for v in read]
        opt.step()
        assert all(v._version > b for v, b in zip(written, before[0])), t
        assert [v._version for v in read] == before[1], t


@pytest.mark.parametrize("scale_grads", [False, True])
def test_clip_adamw_raises_the_version_of_what_it_writes(hip_backend, scale_grads):
    from virconv_amd.optim import ClipAdamW
    ps = [torch.nn.Parameter(rnd((500,), 1)), torch.nn.Parameter(rnd((70,), 2)), torch.nn.Parameter(rnd((9,), 3))]
    opt = ClipAdamW(ps, scale_grads=scale_grads)
    for t in range(3):
        for k, p in enumerate(ps[:2]):
            p.grad = rnd(p.shape, 10 * t + k)
        grads = [p.grad for p in ps[:2]]
        written = ps[:2] + [opt.state[p][k] for p in ps[:2] if p in opt.state for k in ("exp_avg", "exp_avg_sq")]
        written += [opt.total_norm] if opt.total_norm is not None else []
        read = [ps[2]]
        (written if scale_grads else read).extend(grads)
        before = [v._version for v in written], [v._version for v in read]
        opt.step()
        assert all(v._version > b for v, b in zip(written, before[0])), t
        assert [v._version for v in read] == before[1], t


@pytest.mark.parametrize("which", ["AdamW", "ClipAdamW"])
@pytest.mark.parametrize("op", ["norm", "grouped", "torch"])
def test_a_step_between_forward_and_backward_is_refused_by_autograd(hip_backend, op, which):
    from virconv_amd import ops, optim
    x, dy = rnd((30, 24), 1).requires_grad_(), rnd((30, 24), 2)
    w = torch.nn.Parameter(rnd((24,) if op == "norm" else (1, 24, 24) if op == "grouped" else (24, 24), 3))
    offsets = torch.tensor([0, 30], device="cuda")
    run = {"norm": lambda: ops.layer_norm(x, w), "grouped": lambda: ops.grouped_linear(x, w, offsets), "torch": lambda: x @ w}[op]
    opt = getattr(optim, which)([w], lr=1e-3)
    run().backward(dy)
    y = run()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    run().backward(dy)


@pytest.mark.parametrize("which", ["AdamW", "AdamW8", "ClipAdamW"])
def test_the_sparse_bev_stem_follows_its_optimizer(hip_backend, which):
    """The stem keeps its conv weight in a packed form: after every step its map and gradients are those of the dense recipe on the new weight."""
    from test_bev_stem import _backbone_out, _first_block
    from virconv_amd import optim
    from virconv_amd.backbone import HeightCompression
    from virconv_amd.bev_stem import SparseBEVStem
    bd = _backbone_out("cuda")
    t = bd["encoded_spconv_tensor"]
    block = _first_block().cuda().train()
    stem = SparseBEVStem(block)
    assert stem.sparse_path_usable(t)
    opt = {"AdamW": lambda: optim.AdamW(block.parameters(), lr=2e-2), "AdamW8": lambda: optim.AdamW(block.parameters(), lr=2e-2, state_bits=8),
           "ClipAdamW": lambda: optim.ClipAdamW(block.parameters(), lr=2e-2)}[which]()
    pull = rnd((2, 64, 200, 176), 5)
    last = None
    for _ in range(3):
        dense = copy.deepcopy(block)
        opt.zero_grad()
        got = stem(t)
        (got * pull).mean().backward()
        want = dense(HeightCompression({"NUM_BEV_FEATURES": 256})(dict(bd))["spatial_features"])
        (want * pull).mean().backward()
        # (the tolerances that the stem's own tests derive: 1e-4 of the value and of the largest one)
        assert bool(((got - want).abs() <= 1e-4 * want.abs() + 1e-5 * max(1.0, float(want.detach().abs().max()))).all())
        for p, q in zip(block.parameters(), dense.parameters()):
            assert float((p.grad - q.grad).abs().max()) <= 1e-4 * float(q.grad.abs().max())
        assert last is None or float((got - last).detach().abs().max()) > 1e-2     # the step is large enough to be seen
        last = got
        opt.step()


# ---------------------------------------------------------------------------------------------------------------- not finite
BIAS_TILES = [  # (dtype, rows' bounds, inner, outer): the tiles of the weight product, its rows whole and in pieces
    (F32, [0, 5, 300], 40, 48), (BF16, [0, 5, 300], 40, 48), (F16, [0, 9001], 40, 48),          # 64 x 64
    (F32, [0, 5, 300], 200, 328), (BF16, [0, 5, 300], 200, 328), (F16, [0, 5, 300], 200, 328),  # 128 x 128
    (F32, [0, 9001], 136, 264), (BF16, [0, 9001], 136, 264),                                    # ... in pieces
    (BF16, [0, 5, 300], 2560, 4096), (F16, [0, 5, 300], 2560, 2056),                            # 256 x 256
    (F32, [0, 5, 300], 5, 328), (BF16, [0, 5, 300], 5, 328),                                    # few channels
]


@pytest.mark.parametrize("dtype,ends,inner,outer", BIAS_TILES, ids=str)
def test_a_bias_gradient_keeps_undefined_values_in_their_channel(hip_backend, dtype, ends, inner, outer):
    from virconv_amd import ops
    groups, n = len(ends) - 1, ends[-1]
    x, w, b, dy = rnd((n, inner), 1, dtype), rnd((groups, outer, inner), 2, dtype), rnd((groups, outer), 3, dtype), rnd((n, outer), 4, dtype)
    offsets = torch.tensor(ends, device="cuda")

    def run(dy):
        leaves = [w.detach().requires_grad_(), b.detach().requires_grad_()]
        return torch.autograd.grad(ops.grouped_linear(x, leaves[0], offsets, leaves[1]), leaves, dy)

    dw, db = run(dy)
    for value in (math.inf, -math.inf, math.nan):
        for c in (0, 17, outer // 2 + 3, outer - 1):
            bad = dy.clone()
            bad[n - 7, c] = value            # (a row of the last group)
            gw, gb = run(bad)
            keep = torch.ones(outer, dtype=torch.bool, device="cuda")
            keep[c] = False
            assert torch.equal(gb[:-1], db[:-1]) and torch.equal(gb[-1, keep], db[-1, keep]), (value, c)
            assert torch.equal(gw[:-1], dw[:-1]) and torch.equal(gw[-1, keep], dw[-1, keep]), (value, c)
            assert not bool(torch.isfinite(gb[-1, c])) and not bool(torch.isfinite(gw[-1, c]).any()), (value, c)


# ---------------------------------------------------------------------------------------------------------------- operands of few elements
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("few", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("many", [8, 31, 33, 65, 200, 1030])
def test_grouped_linear_with_few_channels_on_one_side(hip_backend, many, few, dtype):
    """Heads of a few outputs, layers of a few inputs: summed axes of several steps, either way."""
    from test_row_ops_gpu import check_grouped
    ends = [2, 40, 40, 41, 230]
    for inner, outer in ((few, many), (many, few)):
        check_grouped(rnd((233, inner), 1, dtype), rnd((4, outer, inner), 2, dtype, inner ** -0.5), ends, rnd((4, outer), 3, dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("few", [1, 4, 7])
def test_grouped_linear_with_few_channels_and_many_rows(hip_backend, few, dtype):
    from test_row_ops_gpu import check_grouped
    ends = [0, 4000, 4001, 4001, 9001]
    for inner, outer in ((few, 72), (72, few), (few, few)):
        check_grouped(rnd((9001, inner), 1, dtype), rnd((4, outer, inner), 2, dtype), ends, rnd((4, outer), 3, dtype), rnd((9001, outer), 4, dtype, 0.1))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_grouped_linear_of_rows_far_apart(hip_backend, dtype):
    """Row strides beyond 32-bit offsets in a tile."""
    from test_row_ops_gpu import check_grouped
    n, inner, outer, stride = 150, 100, 72, (1 << 22) + 8
    x = torch.zeros((n - 1) * stride + inner, dtype=dtype, device="cuda").as_strided((n, inner), (stride, 1))
    x.copy_(rnd((n, inner), 1, dtype))
    check_grouped(x, rnd((3, outer, inner), 2, dtype, 0.1), [0, 70, 70, 150], rnd((3, outer), 3, dtype))


# ---------------------------------------------------------------------------------------------------------------- fp32 products
def one_sided(n, seed):
    """Mantissas whose 16 low bits are nearly all set behind either piece's border, and random ones."""
    g = torch.Generator().manual_seed(seed)
    worst = torch.tensor([1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -16 - 2.0 ** -23, 1 + 2.0 ** -7 - 2.0 ** -15 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23,
                          1 + 2.0 ** -9 - 2.0 ** -17 - 2.0 ** -23, 2 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -17 - 2.0 ** -22, 1.0])
    x = 1 + torch.rand(n, generator=g)
    x[:worst.numel()] = worst
    return x * torch.exp2(torch.randint(-6, 7, (n,), generator=g).float()) * (1 - 2 * torch.randint(0, 2, (n,), generator=g).float())


@pytest.mark.parametrize("inner,outer,rows", [(1, 200, 64), (8, 40, 30), (100, 200, 500), (136, 264, 700), (520, 392, 2600), (4100, 72, 40)])
def test_fp32_products_of_one_term(hip_backend, inner, outer, rows):
    """One product a result (the other operands are zero).  The terms left out stay below u of it.  The six others are added the smallest first; the
    matrix unit cuts what it adds to a larger product at one step of the result, 2 u, which comes once at the product's size and four times at 2^-7 of
    it or less: 3 u + 4 * 2 u / 128 at most."""
    from virconv_amd import ops
    tol = (3 + 2.0 ** -4) * U
    # forward and input gradient: one channel of each row is not zero
    at = torch.arange(rows) % inner
    x = torch.zeros(rows, inner)
    x[torch.arange(rows), at] = one_sided(rows, 1)
    w = one_sided(outer * inner, 2).view(1, outer, inner)
    out_at = torch.arange(rows) % outer
    dy = torch.zeros(rows, outer)
    dy[torch.arange(rows), out_at] = one_sided(rows, 3)
    xc, wc = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = ops.grouped_linear(xc, wc, torch.tensor([0, rows], device="cuda"))
    dx, = torch.autograd.grad(y, xc, dy.cuda())
    for got, want in ((y, x.double()[torch.arange(rows), at][:, None] * w.double()[0][:, at].T),
                      (dx, dy.double()[torch.arange(rows), out_at][:, None] * w.double()[0][out_at])):
        err = (got.detach().double().cpu() - want).abs() / want.abs()
        assert float(err.max()) <= tol, float(err.max()) / U
    # weight gradient: one row of each group is not zero
    groups = 3
    ends = [0, rows // 3, rows // 3 + 1, rows]
    x, dy = torch.zeros(rows, inner), torch.zeros(rows, outer)
    live = [0, rows // 3, rows - 1]
    for k, r in enumerate(live):
        x[r], dy[r] = one_sided(max(inner, 8), 10 + k)[:inner], one_sided(outer, 20 + k)
    wc = torch.zeros(groups, outer, inner, device="cuda", requires_grad=True)
    y = ops.grouped_linear(x.cuda(), wc, torch.tensor(ends, device="cuda"))
    dw, = torch.autograd.grad(y, wc, dy.cuda())
    want = torch.stack([dy[r].double()[:, None] * x[r].double() for r in live])
    err = (dw.double().cpu() - want).abs() / want.abs()
    assert float(err.max()) <= tol, float(err.max()) / U


@pytest.mark.parametrize("rows,inner,outer", [(20, 8, 40), (500, 100, 200)])
def test_fp32_products_at_the_ends_of_the_range(hip_backend, rows, inner, outer):
    """Operands up to the largest number that rounds to a finite bf16; larger ones, infinities and NaN make their results undefined, and no others."""
    from virconv_amd import ops
    offsets = torch.tensor([0, rows], device="cuda")
    w = one_sided(outer * inner, 2).view(1, outer, inner) * 2.0 ** -20
    for size in (2.0 ** 128 - 2.0 ** 119 - 2.0 ** 104, -(2.0 ** 128 - 2.0 ** 120), 3e38, 2.0 ** -100):
        x = torch.zeros(rows, inner)
        x[:, inner // 2] = size
        y = ops.grouped_linear(x.cuda(), w.cuda(), offsets)
        want = x.double() @ w[0].double().T
        assert float(((y.double().cpu() - want).abs() / want.abs()).max()) <= (3 + 2.0 ** -4) * U, size
    x = rnd((rows, inner), 1)
    want = ops.grouped_linear(x, w.cuda(), offsets)
    for size in (2.0 ** 128 - 2.0 ** 119, torch.finfo(F32).min, math.inf, math.nan):
        x[3, inner - 1] = size
        y = ops.grouped_linear(x, w.cuda(), offsets)
        keep = torch.arange(rows, device="cuda") != 3
        assert not bool(torch.isfinite(y[3]).any()) and torch.equal(y[keep], want[keep]), size


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("value", [2e19, 1e25, -3e38])
def test_adamw_8_bit_with_a_square_beyond_fp32(hip_backend, value, dtype):
    """A finite gradient whose square overflows: v is infinite, m / sqrt(v) is 0, and the parameter only decays, as with 32-bit moments."""
    from virconv_amd.optim import AdamW
    wide, narrow, clean = (torch.nn.Parameter(rnd((300,), 1, dtype)) for _ in range(3))
    opts = AdamW([wide], **HYPER), AdamW([narrow], state_bits=8, **HYPER), AdamW([clean], state_bits=8, **HYPER)
    at = torch.tensor([3, 130, 299], device="cuda")
    rest = torch.ones(300, dtype=torch.bool, device="cuda")
    rest[at] = False
    for t in range(4):
        for p in (wide, narrow, clean):
            p.grad = rnd((300,), 10 + t, dtype)
            if t == 1 and p is not clean:
                p.grad[at] = value
        for o in opts:
            o.step()
        assert bool(torch.isfinite(narrow).all()) and bool(torch.isfinite(wide).all()), t
        if t >= 1:
            before = wide_before.float(), narrow_before.float()
            for p, b in zip((wide, narrow), before):
                want = b[at].double() * (1 - HYPER["lr"] * HYPER["weight_decay"])
                assert bool(((p[at].double() - want).abs() <= half_step(dtype) * want.abs() + 3 * U * want.abs() + floor_step(dtype)).all()), t
        wide_before, narrow_before = wide.detach().clone(), narrow.detach().clone()
    # the neighbours: their blocks' exponent of m may differ, by 8-bit roundings then, so steps of lr at most
    assert float((narrow[rest].float() - clean[rest].float()).abs().max()) <= 3 * 4 * HYPER["lr"] + 4 * half_step(dtype) * float(clean.abs().max())


def test_adamw_8_bit_second_moment_settles_where_it_is_said_to(hip_backend):
    """Gaussian gradients of one size for many steps.  A rounding of r to its grid, s apart, adds s |d| to the mean of r^2 where a step changes r by
    d, far less than s: E |d| = (1 - beta2) r E|g^2 / v - 1| / 2 = 0.484 (1 - beta2) r, and what a step adds stays for 1 / (1 - beta2) steps, so v
    settles 0.484 s / r above its mean in 32 bits, s / r between 1/16 and 1/8."""
    from virconv_amd.optim import AdamW
    n, beta2 = 1 << 16, 0.99
    narrow, wide = (torch.nn.Parameter(torch.zeros(n, device="cuda")) for _ in range(2))
    opts = [AdamW([p], lr=0.0, betas=(0.9, beta2), state_bits=b) for p, b in ((narrow, 8), (wide, 32))]
    g = torch.Generator(device="cuda").manual_seed(1)
    ratio = []
    for t in range(900):
        narrow.grad = torch.randn(n, device="cuda", generator=g)
        wide.grad = narrow.grad
        for o in opts:
            o.step()
        if t >= 800:
            ratio.append(float(opts[0].decoded_state(narrow)[1].double().mean() / opts[1].decoded_state(wide)[1].double().mean()))
    excess = sum(ratio) / len(ratio) - 1
    # the estimate's own error: v of one element spreads by sqrt((1 - beta2)) = 10 per cent, of 65536 by 0.04; second-order terms below a tenth of it
    assert 0.484 / 16 * 0.9 - 0.002 < excess < 0.484 / 8 * 1.1 + 0.002, excess


def test_one_row_with_any_stride_through_the_c_interface(hip_backend):
    """A single row's stride means nothing, also where the row is longer than 32-bit offsets into the weights allow."""
    from virconv_amd import _lib
    lib = _lib.load()
    inner, outer = (1 << 24) - 8, 136
    x = torch.zeros(1, inner, device="cuda")
    w = torch.zeros(1, outer, inner, device="cuda")
    x[0, -3:] = torch.tensor([1.0, 2.0, 3.0])
    w[0, :, -3:] = rnd((outer, 3), 1)
    offsets = torch.tensor([0, 1], device="cuda")
    size = lib.vc_grouped_linear_workspace_bytes(0, 1, 1, inner, outer, 0)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    want = (w[0, :, -3:].double() @ x[0, -3:].double()).cpu()
    for stride in (inner, 8, 0):
        y = torch.full((1, outer), math.nan, device="cuda")
        _lib.check(lib.vc_grouped_linear_forward(x.data_ptr(), stride, 1, w.data_ptr(), None, offsets.data_ptr(), 64, 1, inner, outer, 0, y.data_ptr(),
                                                 ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream), "forward")
        torch.cuda.synchronize()
        assert bool(((y[0].double().cpu() - want).abs() <= 8 * U * (w[0, :, -3:].abs().double().cpu() @ x[0, -3:].double().cpu())).all()), stride


# ---------------------------------------------------------------------------------------------------------------- graphs, refusals
@pytest.mark.parametrize("what", ["rows of three axes", "a transposed weight", "a layer in between"])
def test_a_captured_backward_beside_an_eager_graph_is_refused_through_nodes_in_between(hip_backend, what):
    from virconv_amd import ops
    x, dy = rnd((30, 10, 64), 1).requires_grad_(), rnd((30, 10, 64), 3)
    w = rnd((2, 64, 64), 2).requires_grad_()
    scale = rnd((64,), 4).requires_grad_()
    offsets = torch.tensor([0, 100, 300], device="cuda")

    def forward():
        if what == "rows of three axes":
            return ops.layer_norm(x, scale.detach())
        if what == "a transposed weight":
            return ops.grouped_linear(x.detach().view(300, 64), w.transpose(1, 2), offsets).view(30, 10, 64)
        return ops.layer_norm(torch.tanh(x * 2.0), scale.detach())

    leaves = {"rows of three axes": (x,), "a transposed weight": (w,), "a layer in between": (x,)}[what]

    def run():
        y = forward()
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = [t.clone() for t in run()]
    alive = forward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="let go of that result"):
        with torch.cuda.graph(graph):
            run()
    del alive, graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_adamw_counts_the_steps_that_it_took(hip_backend):
    """Parameters of two types, one call each; the second is refused: the first has taken its step, and says so."""
    from virconv_amd.optim import AdamW
    a, b = torch.nn.Parameter(rnd((64,), 1)), torch.nn.Parameter(rnd((64,), 2, BF16))
    twin = torch.nn.Parameter(a.detach().clone())
    opt, alone = AdamW([a, b], **HYPER), AdamW([twin], **HYPER)
    for t in range(4):
        a.grad, b.grad = rnd((64,), 10 + t), rnd((64,), 20 + t, BF16)
        twin.grad = a.grad
        alone.step()
        if t == 2:
            kept = opt.state[b]["exp_avg"]
            opt.state[b]["exp_avg"] = opt.state[b]["exp_avg_sq"]
            before = b.detach().clone()
            with pytest.raises(RuntimeError, match="overlap"):
                opt.step()
            opt.state[b]["exp_avg"] = kept
            assert torch.equal(b, before) and opt.state[b]["step"] == 2
        else:
            opt.step()
        assert torch.equal(a, twin) and opt.state[a]["step"] == t + 1
    assert opt.state[b]["step"] == 3


def test_adamw_with_a_group_without_parameters(hip_backend):
    from virconv_amd.optim import AdamW
    p, q = torch.nn.Parameter(rnd((64,), 1)), torch.nn.Parameter(rnd((64,), 1))
    one, two = AdamW([{"params": []}, {"params": [p], "lr": 1e-2}], **HYPER), AdamW([q], **{**HYPER, "lr": 1e-2})
    for t in range(2):
        p.grad = q.grad = rnd((64,), 2 + t)
        one.step()
        two.step()
        assert torch.equal(p, q)
