"""Layer norm, grouped products and the multi-tensor AdamW step on the GPU against plain 64-bit implementations.

Tolerances are bounds, not fits: u = 2^-24 is half a step of fp32; a sum of k terms in fp32, in whatever order, is off by at most k u times
the sum of the terms' magnitudes; an output of type t adds half a step of t relative to the value."""
import math

import pytest
import torch

from rowref import Adam8, decode_blocks, floor_step, grouped64, half_step, norm64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rnd(shape, seed, dtype=F32, scale=1.0, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(dev)


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = (got - want).abs() > tol
    assert not bool(bad.any()) and bool(torch.isfinite(got).all()), (
        what, int(bad.sum()), float(((got - want).abs() - tol).max()), float((got - want).abs().max()))


# ---------------------------------------------------------------------------------------------------------------- layer norm
def norm_bounds(q, x_type, w_type, b_type, y, grads=None):
    """Bounds of every output.  A row's sums are trees over at most 64 terms a lane and 10 levels (a chain of C / 1024 for the widest rows): 80
    additions and a few more operations, so statistics are off by 128 u: mean by 128 u top, rstd by 64 u relative, and
    xh by d = 128 u (top rstd + 2 |xh|)."""
    d = 128 * U * (q["top"] * q["rstd"] + 2 * q["xh"].abs())
    out = [half_step(x_type) * y.abs() + floor_step(x_type) + (d + 4 * U * q["xh"].abs()) * q["w"].abs() + 4 * U * q["b"].abs()]
    if grads is None:
        return out
    dx, dw, db = grads
    c, g, dy = q["xh"].shape[1], q["g"].abs(), q["dy"].abs()
    h = q["xh"].abs()
    mean_g, mean_gh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    # each term's own roundings, the two means' sums, and xh's error where it enters (in the last term twice)
    e = 128 * U * (g + mean_g + h * mean_gh) + d * mean_gh + h * (g * d).mean(1, keepdim=True)
    out.append(half_step(x_type) * dx.abs() + floor_step(x_type) + q["rstd"] * e + 128 * U * dx.abs())
    k = min(q["xh"].shape[0], 4096) + 64      # the longest chain of additions: a block's rows, then the blocks
    out.append(half_step(w_type) * dw.abs() + floor_step(w_type) + k * U * (dy * h).sum(0) + (dy * d).sum(0))
    out.append(half_step(b_type) * db.abs() + floor_step(b_type) + k * U * dy.sum(0))
    return out


def check_norm(x, w, b, dy, eps=1e-5, rows=None):
    from virconv_amd import ops
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, eps), y), "the pass without gradients gives the same values"
    c = x.shape[-1]
    (ry, rdx, rdw, rdb), q = norm64(x.reshape(-1, c), w, b, eps, dy.reshape(-1, c))
    tol = norm_bounds(q, x.dtype, w.dtype if w is not None else F32, b.dtype if b is not None else F32, ry, (rdx, rdw, rdb))
    within(y.reshape(-1, c), ry, tol[0], "y")
    within(grads[0].reshape(-1, c), rdx, tol[1], "dx")
    k = 1
    if w is not None:
        assert grads[k].dtype == w.dtype
        within(grads[k], rdw, tol[2], "dweight")
        k += 1
    if b is not None:
        within(grads[k], rdb, tol[3], "dbias")


NORM_SIZES = [(1, 1), (3, 2), (5, 3), (1, 4), (7, 5), (300, 7), (64, 8), (33, 9), (1000, 16), (129, 31), (4097, 64), (77, 96), (50, 100),
              (130, 231), (65, 256), (33, 511), (40, 513), (9, 1000), (17, 1024), (5, 1030), (6, 2048), (3, 2500), (4, 4096), (3, 8192), (2, 8200),
              (3, 16384), (2, 16390), (2, 40001)]


@pytest.mark.parametrize("types", [(F32, F32), (F16, F16), (BF16, F32), (BF16, BF16)], ids=str)
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_layer_norm(hip_backend, rows, cols, types):
    xt, wt = types
    x = (rnd((rows, cols), 1, scale=1.5) + rnd((cols,), 2)).to(xt)
    check_norm(x, (1 + rnd((cols,), 3, scale=0.2)).to(wt), rnd((cols,), 4, wt, 0.3), rnd((rows, cols), 5, xt, 0.1))


def test_layer_norm_many_short_rows(hip_backend):
    check_norm(rnd((133_579, 16), 1), 1 + rnd((16,), 2, scale=0.2), rnd((16,), 3), rnd((133_579, 16), 4, scale=0.01))


@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(hip_backend, with_w, with_b):
    check_norm(rnd((70, 48), 1), rnd((48,), 2) if with_w else None, rnd((48,), 3) if with_b else None, rnd((70, 48), 4))


def test_layer_norm_other_shapes_and_strides(hip_backend):
    from virconv_amd import ops
    w, b = 1 + rnd((24,), 1, scale=0.1), rnd((24,), 2)
    wide = rnd((100, 64), 3)
    check_norm(wide[:, 5:29], w, b, rnd((100, 64), 4)[:, 40:])          # column slices, unaligned
    check_norm(wide[:, 5:29][::3], w, b, rnd((34, 24), 4))
    check_norm(rnd((24, 100), 5).t(), w, b, rnd((24, 100), 6).t())      # a transposed matrix
    check_norm(rnd((4, 6, 24), 7), w, b, rnd((4, 6, 24), 8))
    check_norm(rnd((24,), 9), w, b, rnd((24,), 10))
    check_norm(rnd((1, 24), 9).expand(5, 24), w, b, rnd((1, 1), 10).expand(5, 24))
    check_norm(rnd((5, 1), 11).expand(5, 24).contiguous() + 1e-3 * rnd((5, 24), 12), w, b, rnd((5, 24), 13))
    half = rnd((1 + 50 * 24,), 14, F16)[1:].view(50, 24)                # rows that begin at odd multiples of two bytes
    check_norm(half, w.half(), b.half(), rnd((50, 24), 15, F16))
    x = rnd((30, 24), 16)
    assert torch.equal(ops.layer_norm(x, w.repeat_interleave(2)[::2], b), ops.layer_norm(x, w, b))


def test_layer_norm_no_rows(hip_backend):
    from virconv_amd import ops
    x, w, b = rnd((0, 24), 1).requires_grad_(), rnd((24,), 2).requires_grad_(), rnd((24,), 3).requires_grad_()
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 24, device="cuda"))
    assert y.shape == (0, 24) and dx.shape == (0, 24) and not dw.any() and not db.any()


@pytest.mark.parametrize("cols", [5, 64, 4100])
def test_layer_norm_rows_of_one_value_and_large_offsets(hip_backend, cols):
    w, b = 1 + rnd((cols,), 1, scale=0.1), rnd((cols,), 2)
    x = torch.zeros((6, cols), device="cuda")
    x[1] = 3.0
    x[2] = 1e4 + rnd((cols,), 3)
    x[3] = 1e-15 * rnd((cols,), 4)
    x[4] = 1e15 * rnd((cols,), 5)
    x[5] = rnd((cols,), 6)
    check_norm(x, w, b, rnd((6, cols), 7))


def test_layer_norm_undefined_values_stay_in_their_row(hip_backend):
    from virconv_amd import ops
    x = rnd((20, 64), 1)
    want = ops.layer_norm(x)
    x[3, 5], x[7, 0], x[9, 1] = math.nan, math.inf, -math.inf
    got = ops.layer_norm(x)
    keep = torch.ones(20, dtype=torch.bool)
    keep[[3, 7, 9]] = False
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[[3, 7, 9]]).all())


def test_layer_norm_gradient_against_differences(hip_backend):
    from virconv_amd import ops
    # f(t) = sum(y(x + t v) * c): central differences in float64 of the fp32 kernel's values; h balances the two errors: the third derivative
    # times h^2 / 6 and the values' rounding over 2 h
    x, v, c = rnd((40, 48), 1), rnd((40, 48), 2), rnd((40, 48), 3)
    w, b, vw, vb = 1 + rnd((48,), 4, scale=0.2), rnd((48,), 5), rnd((48,), 6), rnd((48,), 7)
    h = 2.0 ** -8
    f = lambda t: (ops.layer_norm(x + t * v, w + t * vw, b + t * vb).double() * c).sum()  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, c)
    slope = sum((a.double() * d).sum() for a, d in zip(grads, (v, vw, vb)))
    # values: 40 x 48 terms of about 1, each off by 300 u at random sign -> sqrt(1920) 300 u / h = 0.2; curvature: every row's function of t has
    # third derivatives of some tens, times h^2 / 6, 40 rows at random sign
    assert abs(float((f(h) - f(-h)) / (2 * h) - slope)) < 0.2 + 40 * 100 * h * h / 6


def test_layer_norm_repeats_bit_for_bit_on_other_streams_and_in_graphs(hip_backend):
    from virconv_amd import ops
    x, w, b, dy = rnd((5000, 64), 1), rnd((64,), 2), rnd((64,), 3), rnd((5000, 64), 4)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def run():
        y = ops.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = [t.clone() for t in run()]
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        for t in out:
            t.zero_()
        with torch.no_grad():
            x.copy_(rnd((5000, 64), 10 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run())), k


def test_layer_norm_beyond_two_to_the_31_elements(hip_backend):
    from virconv_amd import ops
    n, c = 65_600, 32_768
    x = torch.zeros((n, c), dtype=F16, device="cuda")
    x[-3:] = rnd((3, c), 1, F16)
    leaf = x.requires_grad_()
    w, b = rnd((c,), 2, F16), rnd((c,), 3, F16)
    y = ops.layer_norm(leaf, w, b)
    dy = torch.zeros((n, c), dtype=F16, device="cuda")
    dy[-3:] = rnd((3, c), 4, F16)
    dx, = torch.autograd.grad(y, leaf, dy)
    (ry, rdx, _, _), q = norm64(x[-3:], w, b, 1e-5, dy[-3:])
    tol = norm_bounds(q, F16, F16, F16, ry, (rdx, rdx.sum(0), rdx.sum(0)))
    within(y[-3:], ry, tol[0], "y")
    within(dx[-3:], rdx, tol[1], "dx")
    assert torch.equal(y[0], b) and not dx[0].any()


# ---------------------------------------------------------------------------------------------------------------- grouped products
def check_grouped(x, w, ends, b=None, dy=None, index=torch.int32):
    from virconv_amd import ops
    offsets = torch.tensor(ends, dtype=index, device="cuda")
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    y = ops.grouped_linear(leaves[0], leaves[1], offsets, leaves[2] if b is not None else None)
    assert y.dtype == x.dtype and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(ops.grouped_linear(x, w, offsets, b), y)
    dy = rnd((x.shape[0], w.shape[1]), 99, x.dtype) if dy is None else dy
    got = (y, *torch.autograd.grad(y, leaves, dy))
    want, size = grouped64(x, w, ends, b, dy)
    # fp32 products: each within 2^-23 of itself (three exact pieces a side, the terms below 2^-24 left out), the others exact; sums of k terms
    inner, outer, rows = w.shape[2], w.shape[1], max(1, x.shape[0])
    for name, g, r, s, k in zip(("y", "dx", "dw", "db"), got, want, size, (inner + 1, outer, rows, rows)):
        if x.dtype == F32:
            k += 2
        within(g, r, half_step(x.dtype) * r.abs() + floor_step(x.dtype) + (k + 4) * U * s, name)
    return got


GROUPED = [  # ends, inner, outer
    ([0, 1], 1, 1), ([0, 3], 8, 8), ([0, 5, 5, 9], 7, 5), ([0, 0, 0, 17], 16, 24), ([0, 40, 130], 33, 65), ([0, 130, 131, 400], 64, 64),
    ([0, 200, 457], 100, 250), ([0, 517], 250, 129), ([0, 300, 300, 900], 130, 192), ([0, 1, 2, 3, 4, 5, 6, 7, 8], 256, 144),
    ([0, 16, 33, 47], 520, 40), ([0, 1000], 27, 16), ([0, 128, 256, 384], 128, 128), ([0, 150, 170, 480], 300, 200), ([0, 0, 192, 330], 65, 129),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("ends,inner,outer", GROUPED)
def test_grouped_linear(hip_backend, ends, inner, outer, dtype):
    n, groups = ends[-1], len(ends) - 1
    check_grouped(rnd((n, inner), 1, dtype), rnd((groups, outer, inner), 2, dtype, inner ** -0.5), ends, rnd((groups, outer), 3, dtype),
                  index=torch.int64 if groups % 2 else torch.int32)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_grouped_linear_long_inner_axis_and_few_rows(hip_backend, dtype):
    # the inner axis is split and its sums joined; the odd length leaves a short last piece
    check_grouped(rnd((37, 5003), 1, dtype), rnd((3, 70, 5003), 2, dtype, 5003 ** -0.5), [2, 12, 12, 35], rnd((3, 70), 3, dtype))


@pytest.mark.parametrize("dtype", [F32, F16], ids=str)
@pytest.mark.parametrize("ends", [[0, 9001], [0, 4000, 4001, 4001, 9001], [5, 5, 8000]])
def test_grouped_linear_long_groups(hip_backend, dtype, ends):
    # the weight gradient's rows are split into pieces
    n = 9001
    check_grouped(rnd((n, 48), 1, dtype), rnd((len(ends) - 1, 40, 48), 2, dtype), ends, rnd((len(ends) - 1, 40), 3, dtype),
                  rnd((n, 40), 4, dtype, 0.1))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("inner,outer", [(64, 8192), (136, 4104), (1064, 2056), (2056, 1064)])
def test_grouped_linear_large_tiles(hip_backend, inner, outer, dtype):
    # enough aligned work for the large tiles in at least one direction: whole and partial tiles, whole and partial last steps, short and empty groups
    ends = [3, 3, 1030, 1031, 2311, 2700, 2703]
    if inner < 200:
        ends = [e * 3 for e in ends]
    n, groups = ends[-1] + 5, len(ends) - 1
    check_grouped(rnd((n, inner), 1, dtype), rnd((groups, outer, inner), 2, dtype, inner ** -0.5), ends, rnd((groups, outer), 3, dtype),
                  rnd((n, outer), 4, dtype, 0.1))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("inner,outer,ends", [(72, 4096, [0, 1900, 1900, 4160]), (328, 2048, [2, 2500, 2520, 8000]), (256, 256, [0, 131072])])
def test_grouped_linear_tall_and_low_large_tiles(hip_backend, inner, outer, ends, dtype):
    # one column of blocks more than whole rounds of 256-row tiles, and sizes that fill them: either height of the large tiles
    n, groups = ends[-1], len(ends) - 1
    for i, o in ((inner, outer), (outer, inner)):
        check_grouped(rnd((n, i), 1, dtype), rnd((groups, o, i), 2, dtype, i ** -0.5), ends, rnd((groups, o), 3, dtype), rnd((n, o), 4, dtype, 0.1))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("ends", [[0, 200, 456, 456, 9001], [8000, 8000, 8256, 8999, 9001], [0, 1, 258, 8745, 9001]])
def test_grouped_linear_groups_of_one_piece_and_of_many(hip_backend, ends, dtype):
    n = 9001
    check_grouped(rnd((n, 48), 1, dtype), rnd((4, 40, 48), 2, dtype), ends, rnd((4, 40), 3, dtype), rnd((n, 40), 4, dtype, 0.1))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("rows,inner,outer", [(50, 4100, 70), (200, 4100, 130), (600, 2100, 260), (1500, 1030, 136), (2500, 200, 700)])
def test_grouped_linear_every_tile_and_cut(hip_backend, rows, inner, outer, dtype):
    # sizes at which the expected times choose other tiles and numbers of pieces
    ends = [0, rows // 5, rows // 5 + 1, rows - 3, rows]
    check_grouped(rnd((rows, inner), 1, dtype), rnd((4, outer, inner), 2, dtype, inner ** -0.5), ends, rnd((4, outer), 3, dtype),
                  rnd((rows, outer), 4, dtype, 0.1))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("count,inner,outer", [(100, 256, 512), (130, 520, 264)])
def test_grouped_linear_many_long_groups(hip_backend, count, inner, outer, dtype):
    # more groups than a wave has lanes, with work for the large tiles
    g = torch.Generator().manual_seed(4)
    sizes = torch.randint(0, 500, (count,), generator=g)
    sizes[::7] = 0
    ends = [3] + (3 + torch.cumsum(sizes, 0)).tolist()
    n = ends[-1] + 4
    check_grouped(rnd((n, inner), 1, dtype), rnd((count, outer, inner), 2, dtype, inner ** -0.5), ends, rnd((count, outer), 3, dtype),
                  rnd((n, outer), 4, dtype, 0.1))


@pytest.mark.parametrize("op", ["norm", "grouped"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_a_captured_backward_beside_an_eager_graph_of_its_leaves_is_refused(hip_backend, op, accumulate):
    from virconv_amd import ops
    x, w, dy = rnd((300, 64), 1).requires_grad_(), rnd((64,) if op == "norm" else (2, 64, 64), 2).requires_grad_(), rnd((300, 64), 3)
    offsets = torch.tensor([0, 100, 300], device="cuda")

    def run():
        y = ops.layer_norm(x, w) if op == "norm" else ops.grouped_linear(x, w, offsets)
        if accumulate:
            y.backward(dy)
            return y.detach(), x.grad, w.grad
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    want = [t.clone() for t in run()]
    alive = ops.layer_norm(x, w) if op == "norm" else ops.grouped_linear(x, w, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="let go of that result"):
        with torch.cuda.graph(graph):
            run()
    del alive, graph
    torch.cuda.synchronize()
    x.grad, w.grad = torch.zeros_like(x), torch.zeros_like(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        x.grad.zero_(), w.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(torch.equal(a, b) for a, b in zip(run()[:1], want))


def test_two_threads_on_streams_of_their_own(hip_backend):
    import threading
    from virconv_amd import ops

    def work(seed):
        x, dy = rnd((3000, 96), seed).requires_grad_(), rnd((3000, 80), seed + 1)
        nw, w, b = rnd((96,), seed + 2).requires_grad_(), rnd((3, 80, 96), seed + 3).requires_grad_(), rnd((3, 80), seed + 4).requires_grad_()
        offsets = torch.tensor([0, 1000, 1001, 2990], device="cuda")
        y = ops.grouped_linear(ops.layer_norm(x, nw), w, offsets, b)
        return [y.detach(), *torch.autograd.grad(y, (x, nw, w, b), dy)]

    want = {s: work(s) for s in (10, 20)}
    torch.cuda.synchronize()
    bad = []

    def run(seed):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(15):
                    got = work(seed)
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[seed])):
                        bad.append(seed)
        except BaseException as e:      # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=run, args=(s,)) for s in want]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_grouped_linear_many_groups(hip_backend):
    g = torch.Generator().manual_seed(3)
    sizes = torch.randint(0, 9, (200,), generator=g)
    sizes[torch.randint(0, 200, (60,), generator=g)] = 0
    ends = [0] + torch.cumsum(sizes, 0).tolist()
    check_grouped(rnd((ends[-1], 40), 1), rnd((200, 24, 40), 2), ends, rnd((200, 24), 3))


@pytest.mark.parametrize("ends", [[3, 9, 20], [-4, 9, 20], [0, 9, 99], [0, 20, 9], [50, 60, 70], [9, 3, 20], [0, 0, 0], [0, 2 ** 31 - 1, 5]])
@pytest.mark.parametrize("rows", [32, 300])
def test_grouped_linear_rows_of_no_group_and_unsorted_offsets(hip_backend, rows, ends):
    # offsets are cut to a rising sequence within [0, rows]: no content of theirs leads out of the tensors
    check_grouped(rnd((rows, 40), 1), rnd((2, 24, 40), 2), ends, rnd((2, 24), 3))


def test_grouped_linear_no_rows_no_groups(hip_backend):
    from virconv_amd import ops
    w = rnd((2, 24, 40), 2).requires_grad_()
    b = rnd((2, 24), 3).requires_grad_()
    x = rnd((0, 40), 1).requires_grad_()
    y = ops.grouped_linear(x, w, torch.zeros(3, dtype=torch.int32, device="cuda"), b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 24, device="cuda"))
    assert y.shape == (0, 24) and dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == w.shape
    y = ops.grouped_linear(rnd((9, 40), 1), rnd((0, 24, 40), 2), torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert y.shape == (9, 24) and not y.any()


def test_grouped_linear_strides(hip_backend):
    wide, dwide = rnd((200, 100), 1, BF16), rnd((200, 90), 2, BF16)
    w, ends = rnd((2, 33, 41), 3, BF16), [0, 90, 200]
    check_grouped(wide[:, 7:48], w, ends, None, dwide[:, 3:36])
    check_grouped(rnd((41, 200), 4, BF16).t(), rnd((2, 41, 33), 5, BF16).transpose(1, 2), ends, None, rnd((33, 200), 6, BF16).t())
    check_grouped(rnd((1, 41), 7, BF16).expand(200, 41), w, ends, None, rnd((1, 1), 8, BF16).expand(200, 33))
    flat = rnd((1 + 200 * 41,), 9, BF16)[1:].view(200, 41)
    check_grouped(flat, w, ends)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_grouped_linear_undefined_values_stay_where_they_belong(hip_backend, dtype):
    from virconv_amd import ops
    x, w, dy = rnd((300, 45), 1, dtype), rnd((3, 70, 45), 2, dtype), rnd((300, 70), 3, dtype)
    offsets = torch.tensor([10, 100, 200, 290], dtype=torch.int32, device="cuda")

    def run():
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        y = ops.grouped_linear(*leaves, offsets)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = run()
    x[:10] = math.nan       # rows of no group: they enter nothing
    x[290:] = math.inf
    dy[:10] = math.nan
    dy[290:] = -math.inf
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    x[150, 44] = math.nan   # the last channel of a row in group 1; the row behind it begins where an overread would end
    w[2, 69, 44] = math.nan
    y, dx, dw = run()
    rows = torch.ones(300, dtype=torch.bool)
    rows[150] = rows[200:290] = False
    assert torch.equal(y[rows], want[0][rows]) and bool(torch.isnan(y[150]).all())
    assert bool(torch.isnan(y[200:290, 69]).all()) and torch.equal(y[200:290, :69], want[0][200:290, :69])
    assert torch.equal(dx[:200], want[1][:200]) and torch.equal(dx[200:290, :44], want[1][200:290, :44])
    assert torch.equal(dw[[0, 2]], want[2][[0, 2]]) and torch.equal(dw[1, :, :44], want[2][1, :, :44]) and bool(torch.isnan(dw[1, :, 44]).all())


def test_grouped_linear_gradient_against_differences(hip_backend):
    from virconv_amd import ops
    # the product is linear in each argument: a difference quotient has no error of its own but the values' rounding
    x, w, b, c = rnd((60, 40), 1), rnd((2, 30, 40), 2), rnd((2, 30), 3), rnd((60, 30), 4)
    offsets = torch.tensor([0, 25, 60], device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.grouped_linear(leaves[0], leaves[1], offsets, leaves[2]), leaves, c)
    for k, t in enumerate((x, w, b)):
        v = rnd(t.shape, 20 + k)
        args = [[a + s * v if j == k else a for j, a in enumerate((x, w, b))] for s in (1.0, -1.0)]
        f = [(ops.grouped_linear(a[0], a[1], offsets, a[2]).double() * c).sum() for a in args]
        # 1800 values, each a sum of 41 terms of about 1 (and a neighbour's in v), off by 45 u * 41 * 2 at most
        assert abs(float((f[0] - f[1]) / 2 - (grads[k].double() * v).sum())) < 1800 * 45 * 82 * U


@pytest.mark.parametrize("shape", [(700, 96, 200, [0, 300, 300, 700]), (9000, 48, 40, [0, 4000, 9000]), (30, 4100, 64, [0, 14, 30])], ids=str)
def test_grouped_linear_repeats_bit_for_bit_on_other_streams_and_in_graphs(hip_backend, shape):
    from virconv_amd import ops
    n, inner, outer, ends = shape
    groups = len(ends) - 1
    x, w, b = (t.requires_grad_() for t in (rnd((n, inner), 1, BF16), rnd((groups, outer, inner), 2, BF16), rnd((groups, outer), 3, BF16)))
    dy = rnd((n, outer), 4, BF16)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")

    def run():
        y = ops.grouped_linear(x, w, offsets, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):      # other group sizes at every replay: they are read on the device
        for t in out:
            t.zero_()
        cut = sorted(int(v) for v in torch.randint(0, n + 1, (groups - 1,), generator=torch.Generator().manual_seed(k)))
        offsets.copy_(torch.tensor([0, *cut, n], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, run())), k


def test_grouped_linear_beyond_two_to_the_31_elements(hip_backend):
    from virconv_amd import ops
    n, inner, outer = 1_100_000, 2048, 8
    x = torch.zeros((n, inner), dtype=BF16, device="cuda")
    x[-40:] = rnd((40, inner), 1, BF16)
    x.requires_grad_()
    w = rnd((2, outer, inner), 2, BF16, inner ** -0.5).requires_grad_()
    ends = [0, n - 33, n]
    y = ops.grouped_linear(x, w, torch.tensor(ends, device="cuda"))
    dy = torch.zeros((n, outer), dtype=BF16, device="cuda")
    dy[-40:] = rnd((40, outer), 3, BF16)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want, size = grouped64(x[-40:], w, [0, 7, 40], None, dy[-40:])
    for name, g, r, s, k in zip(("y", "dx", "dw"), (y[-40:], dx[-40:], dw), want, size, (inner, outer, 40)):
        within(g, r, half_step(BF16) * r.abs() + floor_step(BF16) + (k + 4) * U * s, name)
    assert not y[:100].any() and not dx[:100].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_grouped_linear_large_tiles_beyond_two_to_the_31_elements(hip_backend, dtype):
    from virconv_amd import ops
    n, inner, outer = 1_100_000, 2048, 512
    x = torch.zeros((n, inner), dtype=dtype, device="cuda")
    x[-40:] = rnd((40, inner), 1, dtype)
    x.requires_grad_()
    w = rnd((2, outer, inner), 2, dtype, inner ** -0.5).requires_grad_()
    y = ops.grouped_linear(x, w, torch.tensor([0, n - 33, n], device="cuda"))
    dy = torch.zeros((n, outer), dtype=dtype, device="cuda")
    dy[-40:] = rnd((40, outer), 3, dtype)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want, size = grouped64(x[-40:], w, [0, 7, 40], None, dy[-40:])
    for name, g, r, s, k in zip(("y", "dx", "dw"), (y[-40:], dx[-40:], dw), want, size, (inner + 2, outer + 2, 42)):
        within(g, r, half_step(dtype) * r.abs() + floor_step(dtype) + (k + 4) * U * s, name)
    assert not y[:-40].any() and not dx[:-40].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_grouped_linear_large_tiles_keep_undefined_values_where_they_belong(hip_backend, dtype):
    """NaN and infinities in one group's rows and in rows of no group: every other group's results as without them, bit for bit."""
    from virconv_amd import ops
    n, inner, outer, ends = 16001, 1032, 2056, [8, 4003, 4003, 9001, 15990]
    offsets = torch.tensor(ends, device="cuda")
    x, w, b, dy = rnd((n, inner), 1, dtype), rnd((4, outer, inner), 2, dtype, inner ** -0.5), rnd((4, outer), 3, dtype), rnd((n, outer), 4, dtype)

    def run(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = ops.grouped_linear(leaves[0], leaves[1], offsets, leaves[2])
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = run(x, dy)
    for bad in (float("nan"), float("inf")):
        xb, dyb = x.clone(), dy.clone()
        for t in (xb, dyb):
            t[:8], t[15990:], t[4003:9001] = bad, bad, bad
        y, dx, dw, db = run(xb, dyb)
        for g, r in ((y, want[0]), (dx, want[1])):
            assert not g[:8].any() and not g[15990:].any()
            assert torch.equal(g[8:4003], r[8:4003]) and torch.equal(g[9001:15990], r[9001:15990])
        for g, r in ((dw, want[2]), (db, want[3])):
            assert not g[1].any()      # (the empty group)
            assert torch.equal(g[0], r[0]) and torch.equal(g[3], r[3]) and not torch.isfinite(g[2]).any()


def test_gradients_are_of_first_order_and_say_so(hip_backend):
    from virconv_amd import ops
    x, w = rnd((20, 24), 1).requires_grad_(), rnd((24,), 2).requires_grad_()
    m, offsets = rnd((2, 16, 24), 3).requires_grad_(), torch.tensor([0, 7, 20], device="cuda")
    for f, leaves in ((lambda: ops.layer_norm(x, w), (x, w)), (lambda: ops.grouped_linear(x, m, offsets), (x, m))):
        first = torch.autograd.grad(f().square().sum(), leaves)
        again = torch.autograd.grad(f().square().sum(), leaves, create_graph=True)      # a graph may be asked for ...
        assert all(torch.equal(a, b) for a, b in zip(first, again)) and all(t.requires_grad for t in again)
        with pytest.raises(RuntimeError, match="first-order"):                         # ... its use is refused, not answered with zeros
            torch.autograd.grad(again[0].sum(), leaves)
    # only what is asked for is computed, and accumulation into .grad works
    y = ops.layer_norm(x, w.detach()) + ops.grouped_linear(x, m.detach(), offsets).sum()
    y.sum().backward()
    assert x.grad is not None and w.grad is None and m.grad is None


# ---------------------------------------------------------------------------------------------------------------- AdamW
HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)


def adam_params(sizes, dtype, seed=0, offset=0):
    out = []
    for k, n in enumerate(sizes):
        n = n if isinstance(n, tuple) else (n,)
        flat = rnd((math.prod(n) + offset,), seed + k, dtype, 0.1)
        out.append(torch.nn.Parameter(flat[offset:].view(n)))
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("sizes,offset", [((5,), 0), ((1, 2, 3, 7, 8, 9), 0), ((4096, 2048, 2047, 2049, (33, 7)), 0), ((1000, 77), 1), ((60_001, (3, 5, 7)) * 40, 0)])
def test_adamw_32_bit_against_64_bits(hip_backend, sizes, offset, dtype):
    from virconv_amd.optim import AdamW
    ps = adam_params(sizes, dtype, offset=offset)
    opt = AdamW(ps, **HYPER)
    lr, (b1, b2), eps, wd = HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]
    for t in range(1, 4):
        before = [(p.detach().double().cpu(), *(opt.state[p][k].double().cpu() if p in opt.state else torch.zeros(p.shape, dtype=torch.float64)
                                                for k in ("exp_avg", "exp_avg_sq"))) for p in ps]
        for k, p in enumerate(ps):
            p.grad = rnd(p.shape, 1000 * t + k, dtype, 10.0 ** (-(k % 4)))
        opt.step()
        for p, (p0, m0, v0) in zip(ps, before):
            g = p.grad.double().cpu()
            m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
            step = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
            # roundings: the two factors' own, two products, a sum (three products for v)
            tm = 3 * U * (b1 * m0.abs() + (1 - b1) * g.abs()) + floor_step(F32)
            tv = 4 * U * v + floor_step(F32)
            within(opt.state[p]["exp_avg"], m, tm, "exp_avg")
            within(opt.state[p]["exp_avg_sq"], v, tv, "exp_avg_sq")
            # the step: m's error relative to what it divides, and eight more roundings (half of v's, root, two factors, sum, quotient, product)
            ts = lr / (1 - b1 ** t) * tm / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps) + 10 * U * step.abs()
            want = p0 * (1 - lr * wd) - step
            within(p, want, half_step(dtype) * want.abs() + floor_step(dtype) + ts + 3 * U * (p0.abs() + step.abs()), "param")
        assert all(opt.state[p]["step"] == t for p in ps)


def test_adamw_is_interchangeable_with_torch(hip_backend):
    from virconv_amd.optim import AdamW
    ps, qs = adam_params([(40, 30), 64], F32), adam_params([(40, 30), 64], F32)
    ours, stock = AdamW(ps, **HYPER), torch.optim.AdamW(qs, **HYPER)
    for t in range(6):
        for k, (p, q) in enumerate(zip(ps, qs)):
            p.grad = rnd(p.shape, 100 * t + k)
            q.grad = p.grad.clone()
        ours.step()
        stock.step()
        if t == 2:      # each goes on from the other's checkpoint
            a, b = ours.state_dict(), stock.state_dict()
            ours, stock = AdamW(ps, **HYPER), torch.optim.AdamW(qs, **HYPER)
            ours.load_state_dict(b)
            stock.load_state_dict(a)
    for p, q in zip(ps, qs):
        # six steps of at most lr (and its decay), each with about a dozen roundings on either side
        assert float((p - q).abs().max()) <= 6 * (24 * U * 2 * HYPER["lr"] + 4 * U * float(p.abs().max()))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_8_bit_bit_for_bit(hip_backend, dtype, offset):
    from virconv_amd.optim import AdamW
    sizes = [1, 7, 8, 127, 128, 129, 2047, 2048, 2049, 5000, (13, 31)]
    ps = adam_params(sizes, dtype, offset=offset)
    opt = AdamW(ps, state_bits=8, seed=5, **HYPER)
    refs = [Adam8(p, k, 5) for k, p in enumerate(ps)]
    for t in range(1, 5):
        for k, (p, r) in enumerate(zip(ps, refs)):
            g = rnd(p.shape, 1000 * t + k) * torch.exp(2 * rnd(p.shape, 77 * t + k)) * 10.0 ** (-2 * (k % 4))
            p.grad = (g * (rnd(p.shape, 5 + k) > -1)).to(dtype)
            r.step(p.grad, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
        opt.step()
        for k, (p, r) in enumerate(zip(ps, refs)):
            st, n = opt.state[p], p.numel()
            for name, want in (("exp_avg", r.m), ("exp_avg_rms", r.r)):
                assert torch.equal(st[name].view(torch.uint8).cpu().reshape(-1), want.view(torch.uint8).reshape(-1)[:n]), (t, k, name)
            assert torch.equal(st["exponents"].cpu(), r.e), (t, k)
            # the step is a product with a reciprocal that is off by 2^-23 at most, of a root that is by as much: 2 * 2 u of it, and the product's own
            # rounding in place of the quotient's; then the parameter's difference is rounded (fp16, bf16: to one of two neighbours)
            step = HYPER["lr"] / (1 - HYPER["betas"][0] ** t) * r.ratio.abs()
            off = (p.detach().cpu().reshape(-1).double() - r.p.double()).abs()
            assert bool((off <= 6 * U * step + (2 * half_step(dtype) * r.p.double().abs() + floor_step(dtype)) * (off > 0)).all()), (t, k, float(off.max()))
            r.p = p.detach().cpu().reshape(-1).clone()
            m, v = opt.decoded_state(p)
            assert torch.equal(m.cpu().reshape(-1), decode_blocks(r.m, r.e[:, 0]).reshape(-1)[:n])
            assert torch.equal(v.cpu().reshape(-1), decode_blocks(r.r, r.e[:, 1]).reshape(-1)[:n] ** 2)


def test_adamw_8_bit_moments_follow_small_changes(hip_backend):
    from virconv_amd.optim import AdamW
    # a second moment without gradients decays by 1 - beta2 a step, far below its grid: its mean over many elements has to follow all the same
    p = torch.nn.Parameter(torch.zeros(1 << 16, device="cuda"))
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), state_bits=8)
    p.grad = 1 + rnd((1 << 16,), 1).abs()
    opt.step()
    m0, v0 = (float(t.double().mean()) for t in opt.decoded_state(p))
    p.grad = torch.zeros_like(p)
    for _ in range(200):
        opt.step()
    m, v = (float(t.double().mean()) for t in opt.decoded_state(p))
    # r is what is unbiased; v = r^2 gains its variance: below 6e-5 of v a step of 1e-3 (the grid's step 1/8, met with probability 5e-4 / (1/8)),
    # 1.2 % over 200 steps; 65536 elements average the rest away to below 1 %
    assert 0.999 ** 200 * 0.99 < v / v0 < 0.999 ** 200 * 1.03
    # m falls by 0.9 a step through the whole range of the block to nothing
    assert abs(m / m0) < 1e-6


def test_adamw_8_bit_undefined_gradients(hip_backend):
    from virconv_amd.optim import AdamW
    a, b = adam_params([300], F32)[0], adam_params([300], F32)[0]
    for p, bad in ((a, False), (b, True)):
        opt = AdamW([p], state_bits=8, **HYPER)
        for t in range(3):
            p.grad = rnd((300,), t)
            if bad and t == 1:
                p.grad[3], p.grad[200] = math.nan, math.inf
            opt.step()
    keep = torch.ones(300, dtype=torch.bool)
    keep[[3, 200]] = False
    assert bool(torch.isnan(b[~keep]).all()) and bool(torch.isfinite(b[keep]).all())
    # the neighbours' exponents may differ (an undefined moment has no part in them), by a rounding of 8-bit states then: steps of lr, not more
    assert float((a[keep] - b[keep]).abs().max()) < 3 * HYPER["lr"]


def test_adamw_checkpoints_resume_bit_for_bit(hip_backend):
    import io
    from virconv_amd.optim import AdamW
    for bits, dtype in ((8, BF16), (8, F32), (32, BF16)):
        def go(ps, opt, steps):
            for t in steps:
                for k, p in enumerate(ps):
                    p.grad = rnd(p.shape, 100 * t + k, dtype)
                opt.step()
        one = adam_params([(40, 30), 200, 3], dtype)
        opt = AdamW(one, state_bits=bits, **HYPER)
        go(one, opt, range(4))
        two = adam_params([(40, 30), 200, 3], dtype)
        first = AdamW(two, state_bits=bits, **HYPER)
        go(two, first, range(2))
        f = io.BytesIO()
        torch.save(first.state_dict(), f)
        f.seek(0)
        second = AdamW(two, state_bits=bits, **HYPER)
        second.load_state_dict(torch.load(f, map_location="cpu", weights_only=True))
        go(two, second, range(2, 4))
        assert all(torch.equal(a, b) for a, b in zip(one, two)), (bits, dtype)


def test_adamw_groups_late_gradients_and_other_orders(hip_backend):
    from virconv_amd.optim import AdamW
    shapes = [(8, 6, 3, 5), (30, 20), (17,)]
    mixed = [torch.nn.Parameter(rnd(s, k).to(memory_format=torch.channels_last) if len(s) == 4 else rnd(s, k)) for k, s in enumerate(shapes)]
    mixed[1] = torch.nn.Parameter(rnd((20, 30), 1).t())
    half = torch.nn.Parameter(rnd((100,), 9, BF16))
    plain = [torch.nn.Parameter(p.detach().clone(memory_format=torch.preserve_format)) for p in mixed]
    ours = AdamW([{"params": mixed[:2]}, {"params": [mixed[2], half], "lr": 1e-2, "weight_decay": 0.0}], **HYPER)
    stock = torch.optim.AdamW([{"params": plain[:2]}, {"params": plain[2:], "lr": 1e-2, "weight_decay": 0.0}], **HYPER)
    for t in range(4):
        for k, (p, q) in enumerate(zip(mixed, plain)):
            if k == 1 and t == 0:
                continue                       # no gradient yet: its steps count from the first one it has
            q.grad = rnd(p.shape, 10 * t + k)
            p.grad = q.grad.clone()            # dense rows, whatever the parameter's order
        half.grad = rnd((100,), t, BF16) if t % 2 else None
        ours.step()
        stock.step()
    for p, q in zip(mixed, plain):
        assert float((p - q).abs().max()) <= 4 * (24 * U * 2e-2 + 4 * U * float(q.abs().max()))
    assert ours.state[mixed[1]]["step"] == 3 and ours.state[half]["step"] == 2


def test_adamw_refusals(hip_backend):
    from virconv_amd.optim import AdamW
    p = torch.nn.Parameter(rnd((64,), 1))
    with pytest.raises(ValueError, match="betas"):
        AdamW([p], betas=(1.0, 0.99))
    with pytest.raises(ValueError, match="lr"):
        AdamW([p], lr=-1.0)
    with pytest.raises(ValueError, match="dense"):
        AdamW([torch.nn.Parameter(rnd((64,), 1)[::2])])
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        AdamW([torch.nn.Parameter(rnd((64,), 1).double())])
    opt = AdamW([p])
    p.grad = rnd((64,), 2)
    opt.step()
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([p], state_bits=8).load_state_dict(opt.state_dict())
    opt.state[p]["exp_avg"] = torch.zeros(63, device="cuda")
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    opt.state[p]["exp_avg"] = p.data
    with pytest.raises(RuntimeError, match="overlap"):
        opt.step()
    opt.state[p]["exp_avg"] = torch.zeros(64, device="cuda")
    before = p.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p, before) and opt.state[p]["step"] == 1


def test_adamw_beyond_two_to_the_31_elements(hip_backend):
    from virconv_amd.optim import AdamW
    n, tail = 2 ** 31 + 5000, 3000
    big = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    with torch.no_grad():
        big[-tail:] = rnd((tail,), 1, BF16)
    small = torch.nn.Parameter(big.detach()[-tail:].clone())
    opts = AdamW([big], **HYPER), AdamW([small], **HYPER)
    big.grad = torch.zeros_like(big)
    for t in range(2):
        small.grad = rnd((tail,), 2 + t, BF16)
        big.grad[-tail:] = small.grad
        for o in opts:
            o.step()
        assert torch.equal(big.detach()[-tail:], small.detach()) and not big.detach()[:-tail].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_types_and_missing_gradients_in_one_group(hip_backend, bits):
    """A group of several types, some parameters without a gradient at some steps or at any: each as in an optimizer of its own."""
    from virconv_amd.optim import AdamW
    kinds = [((40, 7), F32), ((300,), BF16), ((129,), F32), ((64, 3), F16), ((5,), BF16), ((2000,), F32)]
    joint = [torch.nn.Parameter(rnd(s, k, t)) for k, (s, t) in enumerate(kinds)]
    apart = [torch.nn.Parameter(p.detach().clone()) for p in joint]
    opt = AdamW(joint, state_bits=bits, seed=5, **HYPER)
    # (a parameter's random numbers follow from its place in the group: the lone one has as many parameters without gradients in front of it)
    ones = [AdamW([*(torch.nn.Parameter(torch.zeros(1, device="cuda")) for _ in range(k)), p], state_bits=bits, seed=5, **HYPER) for k, p in enumerate(apart)]
    for t in range(5):
        for k, (p, q) in enumerate(zip(joint, apart)):
            p.grad = None if k == 2 or (k == 4 and t in (0, 3)) else rnd(p.shape, 100 * t + k, p.dtype)
            q.grad = p.grad
        opt.step()
        for o in ones:
            o.step()
        for p, q in zip(joint, apart):
            assert torch.equal(p, q)
    assert [opt.state[p]["step"] if p in opt.state else 0 for p in joint] == [5, 5, 0, 5, 3, 5]
    for p, o, q in zip(joint, ones, apart):
        if p in opt.state:
            assert all(torch.equal(a, b) for a, b in zip(opt.decoded_state(p), o.decoded_state(q)))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_many_tensors(hip_backend, bits):
    """More tensors than a launch's table holds, of many sizes: those around the tables' ends as in optimizers of their own."""
    from virconv_amd.optim import AdamW
    g = torch.Generator().manual_seed(1)
    sizes = [int(v) for v in torch.randint(1, 6000, (200,), generator=g)]
    joint = [torch.nn.Parameter(rnd((n,), k)) for k, n in enumerate(sizes)]
    places = [0, 1, 63, 64, 75, 76, 77, 87, 88, 89, 127, 128, 151, 152, 153, 175, 176, 199]
    apart = {k: torch.nn.Parameter(joint[k].detach().clone()) for k in places}
    opt = AdamW(joint, state_bits=bits, seed=3, **HYPER)
    ones = {k: AdamW([*(torch.nn.Parameter(torch.zeros(1, device="cuda")) for _ in range(k)), p], state_bits=bits, seed=3, **HYPER) for k, p in apart.items()}
    for t in range(3):
        for k, p in enumerate(joint):
            p.grad = rnd(p.shape, 1000 * t + k)
            if k in apart:
                apart[k].grad = p.grad
        opt.step()
        for o in ones.values():
            o.step()
        for k in places:
            assert torch.equal(joint[k], apart[k]), k


@pytest.mark.parametrize("channels_last", [False, True])
def test_adamw_looks_its_states_over_at_every_step(hip_backend, channels_last):
    from virconv_amd.optim import AdamW
    p = torch.nn.Parameter(rnd((8, 6, 3, 5), 1))
    if channels_last:
        p = torch.nn.Parameter(p.detach().to(memory_format=torch.channels_last))
    for bits, second in ((32, "exp_avg_sq"), (8, "exp_avg_rms")):
        opt = AdamW([p], state_bits=bits)
        for t in range(2):
            p.grad = rnd(p.shape, t)
            opt.step()
        before = p.detach().clone()
        opt.state[p][second].data = opt.state[p][second].data.flatten()[:7].clone()     # the same tensor object, other memory
        with pytest.raises(ValueError, match=second):
            opt.step()
        assert torch.equal(p, before) and opt.state[p]["step"] == 2


# ---------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("bits", [32, 8])
def test_a_row_network_trains_as_in_64_bits(hip_backend, bits):
    """A pre-norm residual layer with a matrix per class, one gradient and one optimizer step, against the same in float64."""
    from virconv_amd.optim import AdamW
    from virconv_amd.row_layers import GroupedLinear, LayerNorm
    torch.manual_seed(0)
    n, c, hidden, groups = 1500, 48, 80, 3
    ends = [0, 400, 400, 1500]
    mods = torch.nn.ModuleList([LayerNorm(c), GroupedLinear(groups, c, hidden), GroupedLinear(groups, hidden, c)]).cuda()
    x, target = rnd((n, c), 1), rnd((n, c), 2)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    opt = AdamW(mods.parameters(), state_bits=bits, **HYPER)
    before = [p.detach().double().cpu() for p in mods.parameters()]
    h = x + mods[2](torch.nn.functional.silu(mods[1](mods[0](x), offsets)), offsets)
    ((h - target) ** 2).sum().backward()

    ref = [p.clone().requires_grad_() for p in before]
    xd = x.double().cpu()
    y = torch.nn.functional.layer_norm(xd, (c,), ref[0], ref[1], mods[0].eps)
    part = lambda t, w, b: torch.cat([t[i:j] @ w[g].T + b[g] for g, (i, j) in enumerate(zip(ends, ends[1:]))])  # noqa: E731
    hr = xd + part(torch.nn.functional.silu(part(y, ref[2], ref[3])), ref[4], ref[5])
    ((hr - target.double().cpu()) ** 2).sum().backward()
    for p, r in zip(mods.parameters(), ref):
        # sums over 1500 rows behind three products of 48 to 80 terms: (1500 + 4 * 80) u of the magnitudes, which are at most some ten times the
        # gradient's largest entry
        assert float((p.grad.double().cpu() - r.grad).abs().max()) <= 10 * 1900 * U * float(r.grad.abs().max())
    grads = [p.grad.double().cpu() for p in mods.parameters()]
    opt.step()
    lr, eps, wd = HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
    for p, p0, g in zip(mods.parameters(), before, grads):
        # the first step: m / (1 - b1) = g, v / (1 - b2) = g^2
        want = p0 * (1 - lr * wd) - lr * g / (g.abs() + eps)
        within(p, want, 4 * U * p0.abs() + 24 * U * lr, "param")


def test_layer_norm_inside_a_sparse_sequential(hip_backend):
    from virconv_amd import ops
    from virconv_amd.row_layers import LayerNorm
    from virconv_amd.spconv import SparseConvTensor, SparseSequential, SubMConv3d
    idx = torch.stack(torch.meshgrid(torch.arange(2), torch.arange(4), torch.arange(5), torch.arange(6), indexing="ij"), -1).view(-1, 4).int().cuda()
    conv, norm = SubMConv3d(8, 16, 3, bias=False, indice_key="a").cuda(), LayerNorm(16).cuda()
    seq = SparseSequential(conv, norm, torch.nn.ReLU())
    x = SparseConvTensor(rnd((idx.shape[0], 8), 1), idx, [4, 5, 6], 2)
    out = seq(x)
    want = torch.relu(ops.layer_norm(conv(x).features, norm.weight, norm.bias, norm.eps))
    assert torch.equal(out.features, want)
    out.features.sum().backward()
    assert norm.weight.grad is not None and conv.weight.grad is not None
