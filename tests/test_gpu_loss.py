"""FakeApproxCrossEntropy against its definition in 64 bits."""
import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"
IGNORE = -100


def make(shape, seed, dtype=F32, std=1.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=gen) * std).to(dtype)


def targets_of(rows, vocabulary, seed, ignored=0.2):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    t = torch.randint(0, vocabulary, (rows,), device=DEV, generator=gen)
    return torch.where(torch.rand(rows, device=DEV, generator=gen) < ignored, torch.full_like(t, IGNORE), t)


@pytest.fixture(scope="module")
def noisy(pkg):
    t = pkg.synth.table_noisy(3)
    return t, pkg.ops.TruthTable(t)


SIZES = [(1, 4, 1), (1, 32, 5003), (2, 7, 9), (5, 64, 1000), (16, 50, 2049), (17, 20, 3), (70, 33, 257), (129, 64, 5003),
         (300, 48, 16390), (1100, 17, 1025),
         # several pieces of the vocabulary; several runs of rows; both
         (2000, 20, 70001), (16500, 9, 100), (16500, 5, 5000), (3, 20, 70001), (40, 16500, 50)]


def reference(pkg, noisy, x, k, bias, t, reduction, grad_loss):
    xg, kg = ref.Grid(pkg, x), ref.Grid(pkg, k)
    z, off = ref.product(noisy[0], xg, kg)
    if bias is not None:
        z = z + bias.double()
        off = off + 1.01 * ref.E * z.abs()
    rows, bound, p, p_off = ref.loss(z, off, t, IGNORE)
    counted = t != IGNORE
    count = max(1, int(counted.sum()))
    share = counted.double() / (count if reduction == "mean" else 1)
    dz = p.clone()
    dz[torch.arange(len(t), device=DEV), t.clamp(min=0)] -= 1
    share = share * (1.0 if grad_loss is None else grad_loss.double())
    dz_off = (p * p_off + 2 * ref.E * (p + dz.abs())) * share.abs()[:, None] + 4 * ref.E * (dz * share[:, None]).abs()
    grads = ref.dense_gradients(dz * share[:, None], dz_off, xg, kg, x.dtype, k.dtype)
    if reduction == "none":
        loss, off = rows, ref.rounded(rows, bound, F32)
    else:
        loss, off = rows.sum(), bound.sum()
        if reduction == "mean":
            loss, off = loss / count, off / count
        off = ref.rounded(loss, off, F32)
    return loss, off, grads


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("x_dtype,k_dtype", [(F32, F32), (BF16, BF16), (F16, F32)], ids=str)
def test_loss_and_gradients(pkg, noisy, size, x_dtype, k_dtype):
    print("size", size, x_dtype, k_dtype, flush=True)
    rows, depth, vocabulary = size
    reduction = ("mean", "sum", "none")[(rows + vocabulary) % 3]
    x, k = make((rows, depth), 1, x_dtype, 2.0), make((depth, vocabulary), 2, k_dtype)
    bias = make((vocabulary,), 3, (F32, BF16)[rows % 2]) if depth % 2 else None
    t = targets_of(rows, vocabulary, 4)
    grad_loss = None if depth % 3 else make(t.shape if reduction == "none" else (), 5)
    fn = pkg.FakeApproxCrossEntropy(noisy[1], IGNORE)
    loss, off, grads = reference(pkg, noisy, x, k, bias, t, reduction, grad_loss)
    only = fn(x, k, t, bias, reduction)
    ref.check(only, loss, off, "loss")
    got, g = fn.loss_and_gradients(x, k, t, bias, reduction, grad_loss)
    assert torch.equal(got, only)
    for name, a, (want, bound) in zip(g._fields, g, grads):
        if a is not None:
            ref.check(a, want, bound, name)
    assert (g.bias is None) == (bias is None)
    again, one = fn.loss_and_gradients(x, k, t.to(torch.int32), bias, reduction, grad_loss, want=("inputs",))
    assert torch.equal(again, only) and torch.equal(one.inputs, g.inputs) and one.kernel is None and one.bias is None


@pytest.mark.parametrize("rows", [6, 40])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_that_do_not_count(pkg, noisy, rows, reduction):
    fn = pkg.FakeApproxCrossEntropy(noisy[1], IGNORE)
    x, k = make((rows, 16), 1), make((16, 300), 2)
    none = torch.full((rows,), IGNORE, device=DEV)
    loss, g = fn.loss_and_gradients(x, k, none, reduction=reduction)
    assert not loss.any() and not g.inputs.any() and not g.kernel.any()
    # a padded batch: the rows that count have the losses and gradients they have beside any others with the same range
    t = targets_of(rows, 300, 3, 0.0)
    half = torch.cat([t[:rows // 2], none[rows // 2:]])
    full, _ = fn.loss_and_gradients(x, k, t, reduction="none")
    part, g = fn.loss_and_gradients(x, k, half, reduction="none")
    assert torch.equal(part[:rows // 2], full[:rows // 2]) and not part[rows // 2:].any()
    assert not g.inputs[rows // 2:].any() and g.inputs[:rows // 2].any()


@pytest.mark.parametrize("rows", [4, 40])
def test_targets_that_are_no_columns(pkg, noisy, rows):
    fn = pkg.FakeApproxCrossEntropy(noisy[1], IGNORE)
    x, k = make((rows, 16), 1), make((16, 300), 2)
    t = targets_of(rows, 300, 3, 0.0)
    for wrong in (300, -1, 1 << 40, -(1 << 40)):
        bad = t.clone()
        bad[1] = wrong
        loss, g = fn.loss_and_gradients(x, k, bad, reduction="none")
        nan = torch.isnan(loss)
        assert nan[1] and int(nan.sum()) == 1
        # (values outside their grid have no gradient, whatever comes from behind them)
        assert torch.equal(torch.isnan(g.inputs[1]), ref.Grid(pkg, x).inside[1]) and torch.isfinite(g.inputs[0]).all()
        assert torch.equal(torch.isnan(g.kernel), ref.Grid(pkg, k).inside)
        assert torch.isnan(fn(x, k, bad))


@pytest.mark.parametrize("rows", [5, 33])
def test_masked_columns(pkg, noisy, rows):
    """A bias that takes columns out of the vocabulary: the type's lowest value, and -infinity; all of them; one infinite logit."""
    fn = pkg.FakeApproxCrossEntropy(noisy[1], IGNORE)
    x, k = make((rows, 24), 1), make((24, 2100), 2)
    t = targets_of(rows, 100, 3, 0.2)
    part, pg = fn.loss_and_gradients(x, k[:, :100].contiguous(), t, reduction="none")
    for mask in (torch.finfo(F32).min, float("-inf")):
        bias = torch.zeros(2100, device=DEV)
        bias[100:] = mask
        # the kernel's range has to be the same for both
        k2 = k.clone()
        k2[:, 100:] = k[:, :100].min()
        loss, g = fn.loss_and_gradients(x, k2, t, bias, "none")
        # the same logits summed in another order: the sums' bound, twice
        assert (loss - part).abs().max() <= 2 * ref.E * (2100 / 64 + 600 + 8 * float(part.max()))
        assert not g.kernel[:, 100:].any() and not g.bias[100:].any()
        assert torch.isfinite(g.inputs).all()
    every = torch.full((2100,), float("-inf"), device=DEV)
    loss, g = fn.loss_and_gradients(x, k, t, every, "none")
    counted = t != IGNORE
    assert torch.isnan(loss[counted]).all() and not loss[~counted].any() and not g.inputs[~counted].any()


def test_difference_of_the_bias(pkg, noisy):
    """The loss is smooth in the bias: a central difference is off by h^2 / 6 of a third derivative below 1, and by the two losses'
    rounding over 2 h."""
    fn = pkg.FakeApproxCrossEntropy(noisy[1], IGNORE)
    for rows in (3, 50):
        x, k, bias, t = make((rows, 16), 1), make((16, 90), 2), make((90,), 3), targets_of(rows, 90, 4)
        _, g = fn.loss_and_gradients(x, k, t, bias)
        h = 0.02
        for c in (0, 17, 89):
            d = torch.zeros(90, device=DEV)
            d[c] = h
            up, down = fn(x, k, t, bias + d), fn(x, k, t, bias - d)
            noise = 2 * ref.E * (300 + 20 * float(up)) / (2 * h)
            assert abs(float(up.double() - down.double()) / (2 * h) - float(g.bias[c])) <= h * h / 6 + noise + 1e-6


def test_shapes(pkg, noisy):
    fn = pkg.FakeApproxCrossEntropy(noisy[1])
    x, k, t = make((2, 3, 16), 1), make((16, 50), 2), targets_of(6, 50, 3).view(2, 3)
    loss, g = fn.loss_and_gradients(x, k, t, reduction="none")
    flat, f = fn.loss_and_gradients(x.view(6, 16), k, t.view(6), reduction="none")
    assert loss.shape == (2, 3) and g.inputs.shape == (2, 3, 16)
    assert torch.equal(loss.view(6), flat) and torch.equal(g.inputs.view(6, 16), f.inputs) and torch.equal(g.kernel, f.kernel)
    none, g = fn.loss_and_gradients(x[:0], k, t[:0])
    assert float(none) == 0.0 and g.inputs.shape == (0, 3, 16) and not g.kernel.any()
    assert fn(x[:0], k, t[:0], reduction="none").shape == (0, 3)
    with pytest.raises(pkg.InvalidArgumentError):
        fn(x, k, t.view(6))
    with pytest.raises(pkg.InvalidArgumentError):
        fn(x, k, t, reduction="max")
    with pytest.raises(pkg.InvalidArgumentError):
        fn(x, k, t.float())
    with pytest.raises(pkg.InvalidArgumentError):
        fn(x, k[:, :0], t)
    with pytest.raises(pkg.InvalidArgumentError):
        fn(x, k[:5], t)


def test_in_a_graph(pkg, noisy):
    fn = pkg.FakeApproxCrossEntropy(noisy[1], IGNORE)
    for rows in (4, 300):
        x, k, bias, t = make((rows, 32), 1, BF16), make((32, 9000), 2, BF16), make((9000,), 3), targets_of(rows, 9000, 4)
        fn.loss_and_gradients(x, k, t, bias)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss, g = fn.loss_and_gradients(x, k, t, bias)
        for trial in range(4):
            x.copy_(make(x.shape, 50 + trial, BF16))
            t.copy_(targets_of(rows, 9000, 60 + trial))
            want, wg = fn.loss_and_gradients(x, k, t, bias)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(loss, want) and all(torch.equal(a, b) for a, b in zip(g, wg))
