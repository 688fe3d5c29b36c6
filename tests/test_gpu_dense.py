"""FakeApproxDense against its definition in 64 bits: every kind of sizes, types, epilogues, packed kernels, gradients."""
import numpy as np
import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"


def make(shape, seed, dtype=F32, std=1.0, mean=0.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=gen) * std + mean).to(dtype)


@pytest.fixture(scope="module")
def tables(pkg):
    # random entries: T[0][0] is not 0, operands do not commute, sums reach their largest
    return {n: (t, pkg.ops.TruthTable(t)) for n, t in (("noisy", pkg.synth.table_noisy(3)), ("random", pkg.synth.table_random(5)),
                                                       ("asymmetric", pkg.synth.table_asymmetric()), ("exact", pkg.synth.table_exact()))}


SIZES = [
    # rows, depth, columns: few rows by ones, twos, fours, eights and more; depths off the fours; columns off the lanes
    (1, 1, 1), (1, 5, 4), (1, 64, 513), (1, 1024, 4096), (2, 63, 130), (3, 257, 31), (4, 100, 1027), (5, 32, 512), (8, 130, 777),
    (9, 33, 600), (16, 200, 1025),
    # many rows
    (17, 1, 3), (18, 7, 2), (33, 66, 65), (64, 255, 129), (130, 64, 1), (131, 1001, 70), (257, 96, 333), (515, 40, 1030),
    # several runs of rows, the last of few; several pieces of columns
    (16389, 5, 3), (20, 12, 8201), (40, 12, 8201), (3, 9, 16400), (50, 9, 16400),
    # brackets that need 64 bits, at the largest depths
    (2, 20001, 33), (40, 20001, 33), (3, 32764, 20), (35, 32764, 20),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("x_dtype,k_dtype", [(F32, F32), (BF16, F32), (F16, BF16), (BF16, F16)], ids=str)
def test_forward(pkg, tables, size, x_dtype, k_dtype):
    print("size", size, x_dtype, k_dtype, flush=True)
    rows, depth, columns = size
    names = list(ref.ACTIVATIONS)
    activation = names[sum(size) % len(names)]
    name = ("noisy", "random", "asymmetric")[(rows + columns) % 3]
    table, handle = tables[name]
    x, k = make((rows, depth), rows, x_dtype, 1.0, 0.3), make((depth, columns), columns + 1, k_dtype, depth ** -0.5)
    bias = make((columns,), 3, (F32, BF16, F16)[depth % 3]) if columns % 2 else None
    residual = make((rows, columns), 4, x_dtype) if depth % 2 else None
    layer = pkg.FakeApproxDense(handle, activation)
    y, pre = layer.call_and_keep(x, k, bias, residual)
    want, z, y_off, z_off = ref.dense(table, ref.Grid(pkg, x), ref.Grid(pkg, k), bias, residual, activation)
    ref.check(pre, z, ref.rounded(z, z_off, x_dtype), "pre")
    ref.check(y, want, ref.rounded(want, y_off, x_dtype), "output")
    assert torch.equal(layer(x, k, bias, residual), y)
    assert torch.equal(layer(x, layer.pack(k), bias, residual), y)


FEW = [
    # one and two rows: all of the input's codes in a workgroup, and just too many; columns beyond a workgroup a CU, and of several pieces
    (1, 16384, 50), (1, 16385, 20), (2, 8192, 40), (2, 8193, 40), (1, 4100, 4200), (1, 30, 16450), (2, 20, 8210), (2, 1030, 4110),
    # more: parts of one block of the depth and of several, groups of eight rows that end early
    (4, 12, 8201), (6, 4000, 70), (13, 700, 2050), (31, 17, 3000), (32, 2500, 1030), (8, 32764, 24),
]


@pytest.mark.parametrize("size", FEW, ids=str)
@pytest.mark.parametrize("x_dtype", [F32, BF16], ids=str)
def test_few_rows(pkg, tables, size, x_dtype):
    print("size", size, x_dtype, flush=True)
    rows, depth, columns = size
    table, handle = tables["random"]
    x, k = make((rows, depth), rows, x_dtype, 1.0, -0.4), make((depth, columns), columns + 1, BF16, depth ** -0.5)
    bias, residual = make((columns,), 3, F16), make((rows, columns), 4, x_dtype)
    layer = pkg.FakeApproxDense(handle, "gelu")
    y, pre = layer.call_and_keep(x, layer.pack(k), bias, residual)
    want, z, y_off, z_off = ref.dense(table, ref.Grid(pkg, x), ref.Grid(pkg, k), bias, residual, "gelu")
    ref.check(pre, z, ref.rounded(z, z_off, x_dtype), "pre")
    ref.check(y, want, ref.rounded(want, y_off, x_dtype), "output")
    assert torch.equal(layer(x, k, bias, residual), y)


@pytest.mark.parametrize("rows", [1, 2])
def test_nan_in_a_token(pkg, tables, rows):
    """NaN widens no range and has the upper end's code."""
    layer = pkg.FakeApproxDense(tables["noisy"][1])
    x, k = make((rows, 23), 1), make((23, 20), 2)
    n, m = x.clone(), x.clone()
    n[0, 3], m[0, 3] = float("nan"), 1e30
    kept = torch.cat([x.flatten()[:3], x.flatten()[4:]])
    fixed = pkg.FakeApproxDense(tables["noisy"][1], input_minmax=tuple(float(v) for v in kept.aminmax()))
    for kernel in (k, layer.pack(k)):
        assert torch.equal(layer(n, kernel), fixed(m, kernel))


def test_a_range_set_later(pkg, tables):
    layer = pkg.FakeApproxDense(tables["noisy"][1])
    x, k = make((5, 23), 1), make((23, 20), 2)
    own = layer(x, k)
    layer.input_minmax = (-8.0, 8.0)
    wide = layer(x, k)
    assert torch.equal(wide, pkg.FakeApproxDense(tables["noisy"][1], input_minmax=(-8.0, 8.0))(x, k)) and not torch.equal(wide, own)


@pytest.mark.parametrize("rows", [1, 4, 16, 40])
@pytest.mark.parametrize("lo,hi", [(-1.0, 1.0), (0.0, 2.5), (0.5, 3.0), (-4.0, -0.25)])
def test_fixed_range(pkg, tables, rows, lo, hi):
    table, handle = tables["asymmetric"]
    x, k = make((rows, 50), 1, F32, 2.0), make((50, 36), 2)
    layer = pkg.FakeApproxDense(handle, input_minmax=(lo, hi))
    want, _, off, _ = ref.dense(table, ref.Grid(pkg, x, (lo, hi)), ref.Grid(pkg, k))
    for kernel in (k, layer.pack(k)):
        ref.check(layer(x, kernel), want, ref.rounded(want, off, F32))


@pytest.mark.parametrize("rows", [2, 64])
def test_as_the_convolution(pkg, tables, rows):
    """The layer call of a 1x1 convolution has the same codes and sums; its float sums of the operands are rounded otherwise."""
    _, handle = tables["noisy"]
    x, k, bias = make((rows, 48), 7), make((48, 40), 8), make((40,), 9)
    conv = pkg.FakeApproxConv2D((1, 1), handle, "VALID", activation="relu")
    got = pkg.FakeApproxDense(handle, "relu")(x, k, bias)
    want = conv(x.view(1, 1, rows, 48), k.view(1, 1, 48, 40), bias).view(rows, 40)
    # the convolution adds 48 raw values to |m| sums each, in float32, and multiplies by the other's offset (at most 4)
    bound = 48 * 64 * ref.E * (x.abs().sum(1).max() * k.abs().max() + k.abs().sum(0).max() * x.abs().max()).double()
    # raw sums, not sums on the grid: half a step of each operand, 48 times, times the other's offset
    step = (x.max() - x.min()) / 255 * k.abs().max() + (k.max() - k.min()) / 255 * x.abs().max()
    assert (got - want).abs().max() <= bound + 48 * 0.51 * step.double()


def test_shapes_and_strides(pkg, tables):
    table, handle = tables["noisy"]
    layer = pkg.FakeApproxDense(handle)
    for rows in (6, 42):
        wide = make((2, rows // 2, 80), 1)
        x = wide[:, :, 3:67]                                   # rows apart, and off the vectors' alignment
        flat = make((64 * 33 + 1,), 2)[1:].view(64, 33)        # contiguous at an odd float
        turned = make((33, 64), 3).t()                         # columns first
        for k in (flat, turned):
            y = layer(x, k)
            assert y.shape == (2, rows // 2, 33) and y.is_contiguous()
            want, _, off, _ = ref.dense(table, ref.Grid(pkg, x.reshape(rows, 64)), ref.Grid(pkg, k))
            ref.check(y.view(rows, 33), want, ref.rounded(want, off, F32))
        odd = make((rows * 64 + 1,), 4, BF16)[1:].view(rows, 64)   # at an odd halfword
        residual = make((rows * 33 + 1,), 5, BF16)[1:].view(rows, 33)
        y = layer(odd, flat, None, residual)
        want, _, off, _ = ref.dense(table, ref.Grid(pkg, odd), ref.Grid(pkg, flat), None, residual)
        ref.check(y, want, ref.rounded(want, off, BF16))
    assert layer(make((64,), 1), make((64, 7), 2)).shape == (7,)


@pytest.mark.parametrize("rows", [3, 30])
def test_degenerate_operands(pkg, tables, rows):
    table, handle = tables["random"]
    layer = pkg.FakeApproxDense(handle)
    x, k, bias = make((rows, 20), 1), make((20, 9), 2), make((9,), 3)
    zeros = layer(torch.zeros_like(x), k, bias)                # a range of nothing but 0: products are 0
    assert torch.equal(zeros, bias.expand(rows, 9))
    assert torch.equal(layer(x, torch.zeros_like(k), bias), bias.expand(rows, 9))
    assert torch.equal(layer(torch.full_like(x, 3.0), k), torch.zeros(rows, 9, device=DEV))   # as in the convolution
    # NaN counts as the upper end
    n = x.clone()
    n[1, 3] = float("nan")
    m = x.clone()
    m[1, 3] = 1e30
    lo, hi = (torch.cat([x.flatten()[:23], x.flatten()[24:]]).aminmax())
    fixed = pkg.FakeApproxDense(handle, input_minmax=(float(lo), float(hi)))
    assert torch.equal(layer(n, k), fixed(m, k))
    # infinities make the range infinite: nothing finite comes of it, and nothing faults
    n[0, 0] = float("inf")
    assert not torch.isfinite(layer(n, k)).all()


def test_empty(pkg, tables):
    layer = pkg.FakeApproxDense(tables["noisy"][1], "gelu")
    k = make((8, 5), 1)
    assert layer(make((0, 8), 2), k).shape == (0, 5)
    assert layer(make((3, 8), 2), k[:, :0]).shape == (3, 0)
    assert layer(make((3, 8), 2), layer.pack(k[:, :0])).shape == (3, 0)
    g = layer.gradients(make((0, 5), 1), make((0, 8), 2), k, make((0, 5), 3))
    assert g.inputs.shape == (0, 8) and not g.kernel.any() and g.kernel.shape == (8, 5) and not g.bias.any()
    g = layer.gradients(make((3, 0), 1), make((3, 8), 2), k[:, :0], make((3, 0), 3))
    assert not g.inputs.any() and g.inputs.shape == (3, 8) and g.kernel.shape == (8, 0) and g.bias.shape == (0,)


def test_guard_around_outputs(pkg, tables):
    """Rows and columns that end inside a tile or a vector: nothing behind them is written."""
    lib, rows, depth, columns = pkg._lib.load(), 21, 10, 13
    import ctypes
    for dtype, code in ((F32, 0), (BF16, 1)):
        for n in (rows, 3):
            x, k = make((n, depth), 1, dtype), make((depth, columns), 2, dtype)
            desc = pkg._lib.DenseDesc(n, depth, columns, code, code, 0, 0, 0, 0.0, 0.0)
            size = ctypes.c_size_t()
            assert lib.axc_fake_approx_dense_workspace_bytes(ctypes.byref(desc), 0, ctypes.byref(size)) == 0
            ws = torch.empty(size.value, dtype=torch.uint8, device=DEV)
            out, pre = (torch.full((n * columns + 64,), 7.0, dtype=dtype, device=DEV) for _ in range(2))
            stream = torch.cuda.current_stream().cuda_stream
            assert lib.axc_fake_approx_dense(tables["noisy"][1].handle, ctypes.byref(desc), x.data_ptr(), None, k.data_ptr(), None, None,
                                             None, out.data_ptr(), pre.data_ptr(), ws.data_ptr(), size.value, stream) == 0
            assert (out[n * columns:] == 7).all() and (pre[n * columns:] == 7).all()
            grads = [torch.full((m + 64,), 7.0, dtype=dtype, device=DEV) for m in (n * depth, depth * columns, columns)]
            assert lib.axc_fake_approx_dense_gradients_workspace_bytes(ctypes.byref(desc), ctypes.byref(size)) == 0
            ws = torch.empty(size.value, dtype=torch.uint8, device=DEV)
            assert lib.axc_fake_approx_dense_gradients(ctypes.byref(desc), out.data_ptr(), x.data_ptr(), None, k.data_ptr(), None,
                                                       *[g.data_ptr() for g in grads], ws.data_ptr(), size.value, stream) == 0
            for g, m in zip(grads, (n * depth, depth * columns, columns)):
                assert (g[m:] == 7).all() and not (g[:m] == 7).any()


GRADIENT_SIZES = [(1, 1, 1), (3, 5, 2), (17, 40, 33), (64, 64, 64), (128, 128, 128), (129, 130, 127), (200, 31, 515), (515, 333, 70),
                  (1000, 300, 260), (2, 1500, 900)]


@pytest.mark.parametrize("size", GRADIENT_SIZES, ids=str)
@pytest.mark.parametrize("x_dtype,k_dtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F32, BF16)], ids=str)
def test_gradients(pkg, tables, size, x_dtype, k_dtype):
    print("size", size, x_dtype, k_dtype, flush=True)
    rows, depth, columns = size
    activation = list(ref.ACTIVATIONS)[(rows + columns) % 5]
    x, k = make((rows, depth), 1, x_dtype), make((depth, columns), 2, k_dtype)
    pre, gy = make((rows, columns), 3, x_dtype, 2.0), make((rows, columns), 4, x_dtype)
    layer = pkg.FakeApproxDense(tables["noisy"][1], activation)
    got = layer.gradients(gy, x, k, pre if activation else None)
    dz = gy.double()
    off = torch.zeros_like(dz)
    if activation:
        s = ref.slope(pre, activation)
        dz = dz * s
        # a slope is a few operations of float32, whose exponentials' arguments z^2 / 2 or z are rounded
        off = gy.double().abs() * ref.E * (16 + 4 * pre.double().abs() + 4 * pre.double() ** 2)
    wants = ref.dense_gradients(dz, off, ref.Grid(pkg, x), ref.Grid(pkg, k), x_dtype, k_dtype)
    for name, g, (want, bound) in zip(got._fields, got, wants):
        ref.check(g, want, bound, name)
    one = layer.gradients(gy, x, k, pre if activation else None, want=("kernel",))
    assert one.inputs is None and one.bias is None and torch.equal(one.kernel, got.kernel)


def test_gradients_stop_outside_the_grid(pkg, tables):
    lo, hi = -1.0, 1.5
    x, k, gy = make((70, 30), 1), make((30, 20), 2), make((70, 20), 3)
    layer = pkg.FakeApproxDense(tables["noisy"][1], input_minmax=(lo, hi))
    g = layer.gradients(gy, x, k)
    grid = ref.Grid(pkg, x, (lo, hi))
    assert 0.05 < float((~grid.inside).double().mean()) < 0.5
    assert not g.inputs[~grid.inside].any()
    for name, got, (want, bound) in zip(g._fields, g, ref.dense_gradients(gy.double(), torch.zeros_like(gy.double()), grid,
                                                                        ref.Grid(pkg, k), F32, F32)):
        ref.check(got, want, bound, name)


@pytest.mark.parametrize("rows", [3, 20])
def test_gradients_are_differences(pkg, tables, rows):
    """With the exact table the layer is linear from one grid point to the next: a step of the grid changes the outputs by the
    gradient times the step."""
    lo, hi = -2.0, 2.0
    layer = pkg.FakeApproxDense(tables["exact"][1], input_minmax=(lo, hi))
    grid = ref.Grid(pkg, make((rows, 12), 1), (lo, hi))
    x = grid.values.float()
    k = make((12, 9), 2)
    kg = ref.Grid(pkg, k)
    k = kg.values.float()
    w = make((rows, 9), 3)
    g = layer.gradients(w, x, k)
    kg = ref.Grid(pkg, k)
    base = layer(x, k).double()
    # outputs are off by 3 half steps, their differences by twice that, over a step
    for r, c in ((0, 0), (rows - 1, 11), (1, 5)):
        at = float(grid.values[r, c])
        way = -1.0 if at > 0 else 1.0
        moved = x.clone()
        moved[r, c] = (round(at / grid.scale) + way) * grid.scale
        diff = ((layer(moved, k).double() - base) * w).sum() / (way * grid.scale)
        bound = 8 * ref.E * (base.abs() * w.abs()).sum() / grid.scale + 300 * ref.E * (w[r].abs() @ k[c].abs())
        assert abs(float(diff) - float(g.inputs[r, c])) <= float(bound)
    inner = (kg.codes > 3) & (kg.codes < 252)
    for r, c in inner.nonzero()[:3].tolist():
        moved = k.clone()
        moved[r, c] = (int(kg.codes[r, c]) - kg.zero + 1) * kg.scale
        diff = ((layer(x, moved).double() - base) * w).sum() / kg.scale
        bound = 8 * ref.E * (base.abs() * w.abs()).sum() / kg.scale + 300 * ref.E * (w[:, c].abs() @ x[:, r].abs())
        assert abs(float(diff) - float(g.kernel[r, c])) <= float(bound)


def test_in_a_graph_and_on_streams(pkg, tables):
    """Captured calls replayed between eager ones, two graphs captured on one stream, calls on another stream."""
    layer = pkg.FakeApproxDense(tables["noisy"][1], "silu")
    cases = []
    for i, rows in enumerate((4, 70)):
        x, k, gy = make((rows, 96), 10 + i, BF16), make((96, 72), 20 + i, BF16), make((rows, 72), 30 + i, BF16)
        cases.append((x, k, layer.pack(k), gy))

    def step(c):
        x, k, packed, gy = c
        y, pre = layer.call_and_keep(x, k)
        g = layer.gradients(gy, x, k, pre)
        return y, layer(x, packed), g.inputs, g.kernel, g.bias

    for c in cases:
        step(c)
    torch.cuda.synchronize()
    graphs = []
    side = torch.cuda.Stream()
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(c)
        graphs.append((graph, outs))
    for trial in range(4):
        for c in cases:
            c[0].copy_(make(c[0].shape, 100 + trial, BF16))
        wants = [[t.clone() for t in step(c)] for c in cases]
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, outs), want in zip(graphs, wants):
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
    other = [torch.cuda.Stream() for _ in cases]
    got = []
    for s, c in zip(other, cases):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(c))
    torch.cuda.synchronize()
    for g, want in zip(got, wants):
        assert all(torch.equal(a, b) for a, b in zip(g, want))


PINS = [("set_matrix_rows", v) for v in (1, 2, 3)] + [("set_preexpand", v) for v in (1, -1)] + \
    [("set_tile_columns", v) for v in (16, 32, 64)] + [("set_merged_launches", v) for v in (1, -1)]


@pytest.mark.parametrize("pin", PINS, ids=str)
def test_every_form_of_the_sums(pkg, tables, pin):
    """The kernels that make the sums of many rows leave them in order, in parts or turned: the same comes of them."""
    layer = pkg.FakeApproxDense(tables["random"][1], "relu")
    loss = pkg.FakeApproxCrossEntropy(tables["noisy"][1])
    cases = []
    for rows, depth, columns in ((40, 70, 130), (1000, 300, 72), (260, 1024, 96)):
        x, k = make((rows, depth), rows), make((depth, columns), depth)
        t = torch.arange(rows, device=DEV) % columns
        cases.append((x, k, t, layer(x, k), loss.loss_and_gradients(x, k, t, reduction="none")))
    getattr(pkg.ops, pin[0])(pin[1])
    try:
        for x, k, t, y, (l, g) in cases:
            assert torch.equal(layer(x, k), y)
            l2, g2 = loss.loss_and_gradients(x, k, t, reduction="none")
            # (exponentials are summed chunk by chunk: in another order where the sums come in another one)
            assert (l2 - l).abs().max() <= 2 * ref.E * (256 + 8 * float(l.abs().max()))
            for a, b in zip(g2, g):
                assert b is None or (a - b).abs().max() <= 1e-4 * b.abs().max()
    finally:
        getattr(pkg.ops, pin[0])(0)


def test_gradients_of_many_rows(pkg, tables):
    """As many rows as there may be, operands of more than 2^31 elements: the last rows alone, and sums over all of them."""
    rows, depth, columns = 4194176, 520, 3
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1)
    x = torch.randint(-127, 129, (rows, depth), device=DEV, generator=gen, dtype=torch.int16).to(BF16)
    x[0, 0], x[0, 1] = -127, 128           # the grid is the whole numbers
    k, gy = make((depth, columns), 2, BF16), make((rows, columns), 3, BF16)
    layer = pkg.FakeApproxDense(tables["noisy"][1])
    g = layer.gradients(gy, x, k)
    assert x.numel() > 2 ** 31
    kg = ref.Grid(pkg, k)
    for first in (0, rows // 2, rows - 50):
        part = gy[first:first + 50].double()
        want = part @ kg.values.t()
        size = part.abs() @ kg.values.abs().t()
        ref.check(g.inputs[first:first + 50], want, ref.rounded(want, 2.0 ** -7 * size, BF16))
    total, size = torch.zeros((depth, columns), dtype=torch.float64, device=DEV), 0
    for part in range(0, rows, 1 << 18):
        a, b = x[part:part + (1 << 18)].double().t().contiguous(), gy[part:part + (1 << 18)].double()
        total += a @ b
        size = size + a.abs() @ b.abs()
    # float32 sums of 4.2 M terms in 16 384 steps and more of matrix instructions of 32: off by the square root of their number,
    # in steps of the largest partial sum, which is below the sum of the terms' sizes
    ref.check(g.kernel, total * kg.inside, ref.rounded(total, (2.0 ** -7 / 64 + 64 * ref.E) * size, BF16))


def test_far_offsets(pkg, tables):
    """Outputs of more than 2^31 elements: the last rows, against a call on those alone."""
    rows, depth, columns = 262200, 4, 8200
    x, k = make((rows, depth), 1, BF16), make((depth, columns), 2, BF16)
    lo, hi = (float(v) for v in x.float().aminmax())
    layer = pkg.FakeApproxDense(tables["noisy"][1], input_minmax=(lo, hi))
    y = layer(x, k)
    assert y.numel() > 2 ** 31
    for first, last in ((0, 40), (rows - 60, rows), (131000, 131100)):
        assert torch.equal(y[first:last], layer(x[first:last].contiguous(), k))


def test_packed_out_of_line(pkg, tables):
    """Refused on the host: a packed kernel and a range that do not stand where they must."""
    import ctypes
    lib, layer = pkg._lib.load(), pkg.FakeApproxDense(tables["noisy"][1])
    x, packed = make((3, 16), 1), layer.pack(make((16, 8), 2))
    y, ws = torch.empty((3, 8), device=DEV), torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    desc = ctypes.byref(pkg._lib.DenseDesc(3, 16, 8, 0, 0, 0, 0, 0, 0.0, 0.0))

    def call(seen, at):
        return lib.axc_fake_approx_dense(layer.table.handle, desc, x.data_ptr(), seen, None, packed.data.data_ptr() + at, None, None,
                                         y.data_ptr(), None, ws.data_ptr(), ws.numel(), None)

    assert call(None, 64) == pkg._lib.INVALID_ARGUMENT and b"256" in lib.axc_last_error()
    assert call(ws.data_ptr() + 4, 0) == pkg._lib.INVALID_ARGUMENT and b"8-byte" in lib.axc_last_error()
