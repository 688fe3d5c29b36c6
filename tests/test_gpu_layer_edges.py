"""The transformer layers where values, shapes or sizes are at an edge: infinities in places that do not count, operands that are left
out, shapes that only look right, sizes behind what one launch counts."""
import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")


def make(shape, seed, dtype=F32, std=1.0, mean=0.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=gen) * std + mean).to(dtype)


@pytest.fixture(scope="module")
def noisy(pkg):
    return pkg.ops.TruthTable(pkg.synth.table_noisy(3))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", [3, 13, 52, 1283, 4099, 4100])
@pytest.mark.parametrize("dtype", [F32, F16], ids=str)
def test_a_norm_that_nothing_reads(pkg, kind, width, dtype):
    """Without a gradient of y the norm's weight and bias have none, whatever the rows that were normed hold."""
    norm = pkg.ResidualNorm(kind)
    h, block, gh = make((6, width), 1, dtype), make((6, width), 2, dtype), make((6, width), 3, dtype)
    weight, bias, scale = make((width,), 4, dtype), make((width,), 5, dtype), make((width,), 6, dtype)
    h[1, 0], h[3, width - 1] = INF, NAN
    g = norm.gradients(gh, None, h, block, weight, bias, None, scale)
    assert not g.bias.any() and not g.weight.any()
    assert torch.equal(g.x, gh)
    want = gh.double() * scale.double()
    ref.check(g.block, want, ref.rounded(want, 2 * ref.E * want.abs(), dtype))
    g = norm.gradients(gh, None, h, None, weight, bias)
    assert not g.bias.any() and not g.weight.any() and torch.equal(g.x, gh)


GATES = [  # rows' axes, gates' axes, whether that is one gate for each of a number of runs of neighbouring rows
    ((4, 3), (), True), ((4, 3), (1,), True), ((4, 3), (1, 1), True), ((4, 3), (4,), True), ((4, 3), (4, 1), True), ((4, 3), (4, 3), True),
    ((4, 3), (12,), True), ((4, 3), (1, 4, 1), True), ((4, 3), (3,), False), ((4, 3), (1, 3), False), ((4, 3), (2, 1), False),
    ((4, 3), (6,), False), ((4, 3), (3, 4), False), ((4, 3), (2, 2), False), ((4, 3), (2, 4, 1), False), ((4, 3), (0,), False),
    ((1, 3), (3,), True), ((1, 3), (1, 3), True), ((4, 1, 3), (4, 1, 1), True), ((4, 2, 3), (4, 2), True), ((4, 2, 3), (4, 1, 3), False),
    ((4, 2, 3), (4, 2, 1), True), ((4, 2, 3), (1, 2, 1), False), ((12,), (4,), True), ((12,), (4, 1), True), ((12,), (5,), False),
    ((), (), True), ((), (2,), False),
]


@pytest.mark.parametrize("rows,gates,fits", GATES, ids=str)
def test_gates(pkg, rows, gates, fits):
    norm = pkg.ResidualNorm("rms")
    x, block, weight, gate = make(rows + (20,), 1), make(rows + (20,), 2), make((20,), 3), make(gates + (20,), 4)
    gh = make(rows + (20,), 5)
    if not fits:
        with pytest.raises(pkg.InvalidArgumentError):
            norm(x, block, weight, gate=gate)
        with pytest.raises(pkg.InvalidArgumentError):
            norm.gradients(gh, gh, x, block, weight, gate=gate)
        return
    h, y = norm(x, block, weight, gate=gate)
    each = x.numel() // gate.numel()
    want = x.view(-1, 20).double() + block.view(-1, 20).double() * gate.view(-1, 20).double().repeat_interleave(each, 0)
    if len(rows) > 1 and len(gates) == len(rows):            # the same as the product of both
        assert torch.equal(want.view(h.shape), x.double() + block.double() * gate.double())
    ref.check(h.view(-1, 20), want, ref.rounded(want, 3 * ref.E * want.abs() + 2 * ref.E * (want - x.view(-1, 20)).abs(), F32))
    assert norm.gradients(gh, gh, h, block, weight, gate=gate).gate.shape == gate.shape


@pytest.mark.parametrize("rows", [6, 45])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_gradients_of_the_loss_far_apart(pkg, noisy, rows, dtype):
    """A row's gradient is its own: what the loss' gradient is in other rows, however large, does not reach it."""
    fn = pkg.FakeApproxCrossEntropy(noisy)
    x, k, t = make((rows, 16), 1, dtype), make((16, 300), 2, dtype), torch.arange(rows, device=DEV)
    t[5] = -100
    _, plain = fn.loss_and_gradients(x, k, t, reduction="none")
    assert torch.isfinite(plain.inputs).all()
    some = torch.ones(rows, device=DEV)
    some[0], some[1], some[3] = 2.0 ** 100, 2.0 ** -60, 0.0
    _, g = fn.loss_and_gradients(x, k, t, reduction="none", grad_loss=some)
    want = plain.inputs.double() * some.double()[:, None]        # by powers of two: nothing is rounded otherwise
    assert torch.equal(g.inputs.double(), want)
    for bad in (INF, NAN):
        some[0] = bad
        _, g = fn.loss_and_gradients(x, k, t, reduction="none", grad_loss=some)
        assert torch.equal(g.inputs[1:].double(), want[1:])
        assert not torch.isfinite(g.inputs[0][ref.Grid(pkg, x).inside[0]]).any()
    for reduction in ("sum", "mean"):
        for scale in (-4.0, INF, -INF, NAN):
            _, one = fn.loss_and_gradients(x, k, t, reduction=reduction)
            _, g = fn.loss_and_gradients(x, k, t, reduction=reduction, grad_loss=torch.tensor(scale, device=DEV))
            assert not g.inputs[5].any() and one.inputs[0].any()
            if scale == -4.0:
                assert torch.equal(g.inputs, one.inputs * scale) and torch.equal(g.kernel, one.kernel * scale)
            else:
                assert not torch.isfinite(g.inputs[0][ref.Grid(pkg, x).inside[0]]).any()


def test_more_rows_than_threads_of_a_launch(pkg, noisy):
    """2^26 rows and more, a wavefront each: the last rows, against a call on those alone."""
    rows = (1 << 26) + 37
    x, k, bias = make((rows, 1), 1, BF16), make((1, 2), 2), make((2,), 3)
    lo, hi = (float(v) for v in x.float().aminmax())
    layer = pkg.FakeApproxDense(noisy, "relu", input_minmax=(lo, hi))
    y = layer(x, k, bias)
    for first, last in ((0, 40), ((1 << 22) - 20, (1 << 22) + 20), (rows - 60, rows)):
        assert torch.equal(y[first:last], layer(x[first:last].contiguous(), k, bias))
    assert torch.equal(y[-60:], layer(x, layer.pack(k), bias)[-60:])


@pytest.mark.parametrize("rows", [45, 4097, 5003, 16390])
def test_a_range_handed_on_to_many_rows(pkg, noisy, rows):
    """Rows beyond what the workgroups that read a reported range take at once."""
    norm, layer, loss = pkg.ResidualNorm("rms"), pkg.FakeApproxDense(noisy, "silu"), pkg.FakeApproxCrossEntropy(noisy)
    x, weight, k, gy = make((rows, 24), 1, BF16), make((24,), 2), make((24, 40), 3, BF16), make((rows, 40), 4, BF16)
    _, y, seen = norm.call_in_turn(x, None, weight)
    t = torch.arange(rows, device=DEV) % 40
    for kernel in (k, layer.pack(k)):
        assert torch.equal(layer(y, kernel, input_range=seen), layer(y, kernel))
    _, pre = layer.call_and_keep(y, k)
    for a, b in zip(layer.gradients(gy, y, k, pre, input_range=seen), layer.gradients(gy, y, k, pre)):
        assert torch.equal(a, b)
    assert torch.equal(loss(y, k, t, input_range=seen), loss(y, k, t))


def test_parameters(pkg, noisy):
    """Tensors that require a gradient, where torch does not record, and in the calls that make gradients."""
    dense, loss, norm = pkg.FakeApproxDense(noisy), pkg.FakeApproxCrossEntropy(noisy), pkg.ResidualNorm()
    x, k, w, t = make((5, 16), 1), make((16, 30), 2), make((16,), 3), torch.arange(5, device=DEV)
    xp, kp, wp = (torch.nn.Parameter(v) for v in (x, k, w))
    with torch.no_grad():
        assert torch.equal(dense(xp, kp), dense(x, k)) and torch.equal(loss(xp, kp, t), loss(x, k, t))
        assert torch.equal(norm(xp, xp, wp)[1], norm(x, x, w)[1])
    gy = make((5, 30), 4)
    assert torch.equal(dense.gradients(gy, xp, kp).kernel, dense.gradients(gy, x, k).kernel)
    assert torch.equal(loss.loss_and_gradients(xp, kp, t)[1].inputs, loss.loss_and_gradients(x, k, t)[1].inputs)
    assert torch.equal(norm.gradients(x, x, xp, xp, wp).weight, norm.gradients(x, x, x, x, w).weight)
    assert torch.equal(dense(x, dense.pack(kp)), dense(x, k))
    with pytest.raises(pkg.InvalidArgumentError, match="no_grad"):
        dense(x, kp)


@pytest.mark.parametrize("rows,depth,columns,dtype,activation", [(270003, 8, 1001, F32, None), (270003, 8, 1001, BF16, "gelu"),
                                                                 (360000, 700, 12, BF16, None)], ids=str)
def test_gradients_in_runs_of_rows(pkg, noisy, rows, depth, columns, dtype, activation):
    """More values of the gradient, or of the input, than stand in front of the products at a time."""
    assert rows * (max(depth, columns) + 127) // 128 * 128 > 1 << 28
    x, k, gy = make((rows, depth), 1, dtype), make((depth, columns), 2, dtype), make((rows, columns), 3, dtype)
    pre = make((rows, columns), 4, dtype, 2.0) if activation else None
    lo, hi = (float(v) for v in x.float().aminmax())
    layer = pkg.FakeApproxDense(noisy, activation, input_minmax=(lo, hi))
    g = layer.gradients(gy, x, k, pre)
    # (a product alone may be made by another number of wavefronts a tile: summed in another order, held to the same bounds)
    alone = [getattr(layer.gradients(gy, x, k, pre, want=(one,)), one) for one in ("inputs", "kernel", "bias")]
    ranges = ((0, 200), (261900, 262300), (rows - 300, rows))
    for first, last in ranges:                    # (262144: where runs of 1024 values a row end)
        part = gy[first:last], x[first:last].contiguous(), pre[first:last].contiguous() if activation else None
        few = layer.gradients(part[0].contiguous(), part[1], k, part[2], want=("inputs",)).inputs
        size = gy[first:last].double().abs() @ k.double().abs().t().contiguous()
        # the same terms, summed in another order, of columns + 300 operations, and rounded once each
        for got in (g.inputs, alone[0]):
            off = (got[first:last].double() - few.double()).abs()
            assert (off <= 3 * ref.E * 1.13 * (columns + 300) * size * 1.02 + 2 * ref.half_step(dtype) * few.double().abs()).all()
    total, size, sums, sizes = 0.0, 0.0, 0.0, 0.0
    xg, kg = ref.Grid(pkg, x, (lo, hi)), ref.Grid(pkg, k)
    for r in range(0, rows, 1 << 16):
        dz = gy[r:r + (1 << 16)].double()
        if activation:
            dz = dz * ref.slope(pre[r:r + (1 << 16)], activation)
        a = xg.values[r:r + (1 << 16)].t().contiguous()
        total, size = total + a @ dz, size + a.abs() @ dz.abs()
        sums, sizes = sums + dz.sum(0), sizes + dz.abs().sum(0)
    # float32 sums over all rows: off by the square root of their number, in half steps of sums below the terms' sizes (600 for 360 000);
    # terms are 16 bits or more, slopes of float32 are off by 64 half steps
    for kernel, bias in ((g.kernel, g.bias), alone[1:]):
        ref.check(kernel, total * kg.inside, ref.rounded(total, (2.0 ** -16 / 64 + 600 * ref.E) * size, dtype), "kernel")
        ref.check(bias, sums, ref.rounded(sums, 600 * ref.E * sizes, dtype), "bias")
