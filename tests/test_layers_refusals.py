"""What the transformer layers refuse, without a GPU: descriptions and pointers through the C ABI, tensors through Python."""
import ctypes

import pytest
import torch


def dense(pkg, rows=4, depth=8, columns=8, types=(0, 0, 0), activation=0):
    return pkg._lib.DenseDesc(rows, depth, columns, *types, activation, 0, 0.0, 0.0)


def norm(pkg, rows=4, width=8, groups=0, types=(0, 0), kind=0, eps=1e-6):
    return pkg._lib.ResidualNormDesc(rows, width, groups, *types, kind, eps)


BAD_DENSE = [dict(rows=-1), dict(columns=-1), dict(depth=0), dict(depth=-3), dict(depth=32768), dict(depth=32765), dict(rows=1 << 31),
             dict(columns=1 << 31), dict(rows=1 << 21, columns=1 << 20), dict(types=(3, 0, 0)), dict(types=(0, -1, 0)),
             dict(types=(0, 0, 9)), dict(activation=5), dict(activation=-1)]


@pytest.mark.parametrize("bad", BAD_DENSE, ids=str)
def test_dense_descriptions(pkg, bad):
    lib, n = pkg._lib.load(), ctypes.c_size_t()
    desc = ctypes.byref(dense(pkg, **bad))
    for call in (lambda: lib.axc_dense_packed_bytes(desc, ctypes.byref(n)),
                 lambda: lib.axc_fake_approx_dense_workspace_bytes(desc, 0, ctypes.byref(n)),
                 lambda: lib.axc_fake_approx_dense_gradients_workspace_bytes(desc, ctypes.byref(n)),
                 lambda: lib.axc_fake_approx_cross_entropy_workspace_bytes(desc, 1, ctypes.byref(n)),
                 lambda: lib.axc_dense_pack(desc, 256, 256, None),
                 lambda: lib.axc_fake_approx_dense_gradients(desc, *[256] * 9, 1 << 30, None)):
        assert call() == pkg._lib.INVALID_ARGUMENT
        assert lib.axc_last_error()


def test_dense_arguments(pkg):
    lib, bad, n = pkg._lib.load(), pkg._lib.INVALID_ARGUMENT, ctypes.c_size_t()
    desc = ctypes.byref(dense(pkg))
    assert lib.axc_dense_packed_bytes(None, ctypes.byref(n)) == bad
    assert lib.axc_dense_packed_bytes(desc, None) == bad
    assert lib.axc_fake_approx_dense_workspace_bytes(desc, 0, None) == bad
    assert lib.axc_fake_approx_dense(None, desc, *[256] * 9, 1 << 30, None) == bad
    assert lib.axc_fake_approx_cross_entropy(None, desc, *[256] * 5, -100, 2, *[256] * 6, 1 << 30, None) == bad
    assert lib.axc_dense_pack(desc, None, 256, None) == bad
    assert lib.axc_dense_pack(desc, 256, 260, None) == bad                                     # alignment
    # gradients: tensors, what the activation was given, the workspace
    args = [256] * 9
    assert lib.axc_fake_approx_dense_gradients(desc, None, *args[1:], 1 << 30, None) == bad
    assert lib.axc_fake_approx_dense_gradients(ctypes.byref(dense(pkg, activation=2)), 256, 256, None, 256, None, *args[5:], 1 << 30,
                                               None) == bad
    assert lib.axc_fake_approx_dense_gradients(desc, *args, 16, None) == bad
    assert b"workspace" in lib.axc_last_error()
    assert lib.axc_fake_approx_dense_gradients(desc, *args[:8], None, 1 << 30, None) == bad
    assert lib.axc_fake_approx_dense_gradients(desc, *args[:8], 300, 1 << 30, None) == bad
    many = ctypes.byref(dense(pkg, rows=4194177))
    assert lib.axc_fake_approx_dense_gradients_workspace_bytes(many, ctypes.byref(n)) == pkg._lib.UNIMPLEMENTED
    assert lib.axc_fake_approx_cross_entropy_workspace_bytes(many, 0, ctypes.byref(n)) == pkg._lib.UNIMPLEMENTED


BAD_NORM = [dict(rows=-1), dict(width=0), dict(groups=-1), dict(groups=3), dict(groups=8), dict(types=(3, 0)), dict(types=(0, 3)),
            dict(kind=2), dict(eps=-1.0), dict(eps=float("nan")), dict(rows=1 << 40)]


@pytest.mark.parametrize("bad", BAD_NORM, ids=str)
def test_norm_descriptions(pkg, bad):
    lib, n, tensors = pkg._lib.load(), ctypes.c_size_t(), pkg._lib.ResidualNormTensors(*[256] * 7)
    desc, t = ctypes.byref(norm(pkg, **bad)), ctypes.byref(tensors)
    assert lib.axc_residual_norm_gradients_workspace_bytes(desc, ctypes.byref(n)) == pkg._lib.INVALID_ARGUMENT
    assert lib.axc_residual_norm(desc, t, 256, 256, None, None) == pkg._lib.INVALID_ARGUMENT
    assert lib.axc_residual_norm_gradients(desc, t, 256, 256, 256, t, 256, 1 << 30, None) == pkg._lib.INVALID_ARGUMENT


def test_norm_arguments(pkg):
    lib, bad, T = pkg._lib.load(), pkg._lib.INVALID_ARGUMENT, pkg._lib.ResidualNormTensors
    desc, gated = ctypes.byref(norm(pkg)), ctypes.byref(norm(pkg, groups=2))
    def call(tensors, d=desc, h=256, y=256, seen=None):
        return lib.axc_residual_norm(d, ctypes.byref(tensors), h, y, seen, None)
    x, b, w = 256, 512, 768
    assert call(T(None, b, w)) == bad and call(T(x, b, None)) == bad
    assert call(T(x, None, w, None, None, 256, None)) == bad and call(T(x, None, w, None, None, None, 256)) == bad
    assert call(T(x, b, w, None, 256)) == bad and call(T(x, b, w), gated) == bad        # a gate and its groups
    assert call(T(x, b, w), h=None) == bad and call(T(x, b, w), y=None) == bad and call(T(x, b, w), seen=4) == bad
    wide = ctypes.byref(norm(pkg, width=32769))
    assert call(T(x, b, w), wide) == pkg._lib.UNIMPLEMENTED
    def back(tensors, out, h=256, gh=256, gy=256, ws=256, size=1 << 30):
        return lib.axc_residual_norm_gradients(desc, ctypes.byref(tensors), h, gh, gy, ctypes.byref(out), ws, size, None)
    whole = T(256, 256, 256)
    assert back(T(x, b, w), whole, h=None) == bad and back(T(x, b, w), whole, gh=None, gy=None) == bad
    assert back(T(x, b, w), T(None, 256, 256)) == bad and back(T(x, b, w), T(256, None, 256)) == bad
    assert back(T(x, b, w), T(256, 256, 256, 256)) == bad                                # the gradient of no bias
    assert back(T(x, b, w), whole, size=8) == bad and back(T(x, b, w), whole, ws=8) == bad


def test_python(pkg):
    Invalid, No = pkg.InvalidArgumentError, pkg.UnimplementedError
    with pytest.raises(No):
        pkg.ResidualNorm("batch")
    with pytest.raises(Invalid):
        pkg.ResidualNorm("rms", -1.0)
    with pytest.raises(Invalid):
        pkg.ResidualNorm("rms", float("inf"))
    with pytest.raises(No):
        pkg.FakeApproxDense(None, "tanh")
    with pytest.raises(Invalid):
        pkg.FakeApproxDense(None, num_bits=4)
    with pytest.raises(Invalid):
        pkg.FakeApproxCrossEntropy(None, num_bits=4)
    n = pkg.ResidualNorm()
    x = torch.zeros(2, 4)
    with pytest.raises(Invalid):
        n(x, x, x[0])                       # not on the GPU
    with pytest.raises(Invalid):
        n(3.0, x, x[0])


def test_empty_calls_do_nothing(pkg):
    lib = pkg._lib.load()
    T = pkg._lib.ResidualNormTensors
    assert lib.axc_residual_norm(ctypes.byref(norm(pkg, rows=0)), ctypes.byref(T(None, None, 256)), None, None, None, None) == 0
    n = ctypes.c_size_t(5)
    assert lib.axc_fake_approx_dense_gradients_workspace_bytes(ctypes.byref(dense(pkg, rows=0)), ctypes.byref(n)) == 0
    assert n.value == 0


def test_no_rows_have_no_block(pkg):
    """The tensors of a call without rows hold nothing, and may stand nowhere."""
    lib = pkg._lib.load()
    T = pkg._lib.ResidualNormTensors
    assert lib.axc_residual_norm(ctypes.byref(norm(pkg, rows=0)), ctypes.byref(T(None, None, 256, None, None, 256, 256)), None, None,
                                 None, None) == 0


def test_ranges_out_of_line(pkg):
    """A range is read as pairs of floats."""
    lib, bad = pkg._lib.load(), pkg._lib.INVALID_ARGUMENT
    desc = ctypes.byref(dense(pkg))
    assert lib.axc_fake_approx_dense_gradients(desc, 256, 256, 260, *[256] * 6, 1 << 30, None) == bad
    assert b"8-byte" in lib.axc_last_error()


def test_tensors_that_require_a_gradient(pkg):
    """Refused ahead of all else while torch records: the output would be a constant to it."""
    table = object.__new__(pkg.TruthTable)
    dense, loss, norm = pkg.FakeApproxDense(table), pkg.FakeApproxCrossEntropy(table), pkg.ResidualNorm()
    x, k, w, t = torch.zeros(2, 4), torch.zeros(4, 3), torch.zeros(4), torch.zeros(2, dtype=torch.int64)
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: dense(leaf(x), k), lambda: dense(x, leaf(k)), lambda: dense(x, k, leaf(w[:3])), lambda: dense.call_and_keep(x, leaf(k)),
             lambda: dense(x, k, None, leaf(x[:, :3])), lambda: loss(leaf(x), k, t), lambda: loss(x, leaf(k), t),
             lambda: loss(x, k, t, leaf(w[:3])), lambda: norm(leaf(x), x, w), lambda: norm(x, leaf(x), w), lambda: norm(x, x, leaf(w)),
             lambda: norm.call_in_turn(x, x, w, scale=leaf(w)), lambda: norm(x, x, w, gate=leaf(w))]
    for call in calls:
        with pytest.raises(pkg.InvalidArgumentError, match="no_grad"):
            call()
        with torch.no_grad(), pytest.raises(pkg.InvalidArgumentError, match="on the GPU"):
            call()


@pytest.mark.parametrize("types", [(0, 0, 0), (1, 1, 1), (2, 2, 2)], ids=str)
def test_the_gradients_workspace_is_bounded(pkg, types):
    """Whatever the rows are: copies of 2^28 values of the gradient or of the input, at most three terms of two bytes, straight and
    turned, and what is the kernel's; a 32nd of the gradient for the bias, in float32 by 64 rows; partial sums of two products' 512 tiles
    of 64 KiB where a depth is split."""
    lib, n = pkg._lib.load(), ctypes.c_size_t()
    for rows, depth, columns in ((65536, 4096, 14336), (1 << 20, 4096, 4096), (4194176, 520, 3), (1 << 20, 8192, 64), (300, 32764, 32000)):
        for activation in (0, 2):
            desc = dense(pkg, rows, depth, columns, types, activation)
            assert lib.axc_fake_approx_dense_gradients_workspace_bytes(ctypes.byref(desc), ctypes.byref(n)) == 0
            kernel = (depth + 128) * (columns + 128)
            assert n.value <= (1 << 28) * 2 * (3 + 3 + 1) + kernel * (2 + 4 * 4) + (rows // 64 + 2) * (columns + 128) * 4 + (1 << 26)
