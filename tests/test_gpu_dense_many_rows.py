"""FakeApproxDense of more rows than few_rows_kernel takes, whatever that limit is: operands of no width, NaN, infinities, and what lies
around the outputs of every kernel that makes them."""
import ctypes
import os
import re

import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"


def _few_rows_most():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tf-approximate_amd", "csrc", "layers_api.hip")
    with open(path) as f:
        return int(re.search(r"kFewRowsMost = (\d+);", f.read()).group(1))


FEW = _few_rows_most()
MANY = FEW + 13           # neither a multiple of four nor of a tile
ROWS = [1, 3, FEW, FEW + 1, MANY, 10 * MANY]


def make(shape, seed, dtype=F32, std=1.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=gen) * std).to(dtype)


@pytest.fixture(scope="module")
def table(pkg):
    return pkg.synth.table_random(5)


@pytest.fixture(scope="module")
def handle(pkg, table):
    return pkg.ops.TruthTable(table)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("packed", [False, True])
def test_operands_of_no_width(pkg, handle, rows, packed):
    layer = pkg.FakeApproxDense(handle)
    x, k, bias = make((rows, 20), 1), make((20, 9), 2), make((9,), 3)
    call = lambda x, k, *more: layer(x, layer.pack(k) if packed else k, *more)  # noqa: E731
    assert torch.equal(call(torch.zeros_like(x), k, bias), bias.expand(rows, 9))
    assert torch.equal(call(x, torch.zeros_like(k), bias), bias.expand(rows, 9))
    assert torch.equal(call(torch.full_like(x, 3.0), k), torch.zeros(rows, 9, device=DEV))      # as in the convolution
    assert torch.equal(call(x, torch.full_like(k, -0.25)), torch.zeros(rows, 9, device=DEV))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_nan_and_infinities(pkg, handle, rows, dtype):
    layer = pkg.FakeApproxDense(handle)
    x, k = make((rows, 23), 1, dtype), make((23, 20), 2, dtype)
    at = (rows // 2, 3)
    n, m = x.clone(), x.clone()
    n[at], m[at] = float("nan"), 1e30
    keep = torch.ones(x.shape, dtype=torch.bool, device=DEV)
    keep[at] = False
    fixed = pkg.FakeApproxDense(handle, input_minmax=tuple(float(v) for v in x[keep].float().aminmax()))
    for kernel in (k, layer.pack(k)):
        assert torch.equal(layer(n, kernel), fixed(m, kernel))         # NaN counts as the upper end
    w, v = k.clone(), k.clone()
    w[5, 7] = float("nan")
    kept = torch.ones(k.shape, dtype=torch.bool, device=DEV)
    kept[5, 7] = False
    v[5, 7] = k[kept].max()
    got, want = layer(x, w), layer(x, v)                                # (the grid's upper end and the largest value have one code)
    assert torch.equal(got, want)
    n[0, 0] = float("inf")                                             # nothing finite comes of an infinite range, and nothing faults
    assert not torch.isfinite(layer(n, k)).all()
    n[0, 0] = float("-inf")
    assert not torch.isfinite(layer(n, layer.pack(k))).all()


# dense_out_parts_kernel: few rows; dense_out_kernel: sums in order or in parts; dense_out_turned_kernel of 16 and of 64 columns: sums of
# exchanged operands, fewer than 1024 tiles of 64 x 64 and more
GUARDED = [(3, 10, 13), (FEW, 130, 67), (FEW + 1, 10, 13), (MANY, 130, 67), (130, 64, 1), (387, 101, 1531), (1000, 300, 77),
           (2113, 70, 2051), (4099, 1024, 1027)]


@pytest.mark.parametrize("size", GUARDED, ids=str)
@pytest.mark.parametrize("dtype,code", [(F32, 0), (BF16, 1)], ids=str)
@pytest.mark.parametrize("pin", [None, ("set_matrix_rows", 1), ("set_matrix_rows", 3), ("set_preexpand", 1)], ids=str)
def test_guard_around_outputs(pkg, handle, table, size, dtype, code, pin):
    """What lies in front of the outputs and behind them stays, and all of them is written."""
    lib, (rows, depth, columns) = pkg._lib.load(), size
    x, k, bias = make((rows, depth), 1, dtype), make((depth, columns), 2, dtype), make((columns,), 3)
    residual = make((rows, columns), 4, dtype)
    n, front = rows * columns, 64
    stream = torch.cuda.current_stream().cuda_stream
    if pin:
        getattr(pkg.ops, pin[0])(pin[1])
    try:
        desc = pkg._lib.DenseDesc(rows, depth, columns, code, code, 0, 1, 0, 0.0, 0.0)
        size = ctypes.c_size_t()
        assert lib.axc_fake_approx_dense_workspace_bytes(ctypes.byref(desc), 0, ctypes.byref(size)) == 0
        ws = torch.empty(size.value, dtype=torch.uint8, device=DEV)
        out, pre = (torch.full((front + n + 64,), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
        at = front * out.element_size()
        assert lib.axc_fake_approx_dense(handle.handle, ctypes.byref(desc), x.data_ptr(), None, k.data_ptr(), None, bias.data_ptr(),
                                         residual.data_ptr(), out.data_ptr() + at, pre.data_ptr() + at, ws.data_ptr(), size.value,
                                         stream) == 0
        torch.cuda.synchronize()
    finally:
        if pin:
            getattr(pkg.ops, pin[0])(0)
    for t in (out, pre):
        assert torch.isnan(t[:front]).all() and torch.isnan(t[front + n:]).all() and torch.isfinite(t[front:front + n]).all()
    part = slice(max(0, rows - 70), rows)                              # the last tile's rows
    want, z, y_off, z_off = ref.dense(table, _part(ref.Grid(pkg, x), part), ref.Grid(pkg, k), bias, residual[part], "relu")
    ref.check(pre[front:front + n].view(rows, columns)[part], z, ref.rounded(z, z_off, dtype), "pre")
    ref.check(out[front:front + n].view(rows, columns)[part], want, ref.rounded(want, y_off, dtype), "output")


def _part(grid, rows):
    grid.codes, grid.values, grid.inside = grid.codes[rows], grid.values[rows], grid.inside[rows]
    return grid
