"""How exact the transformer layers' results are, beyond what their sizes alone show: bounds that leave no room for a rounding to fewer
bits on the way than the outputs' type has."""
import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"


def make(shape, seed, dtype=F32, std=1.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=gen) * std).to(dtype)


@pytest.fixture(scope="module")
def noisy(pkg):
    return pkg.ops.TruthTable(pkg.synth.table_noisy(3))


def products(dz, dz_off, xg, kg, x_dtype, k_dtype):
    """((gradient, bound) of the input, of the kernel): the gradient dz goes into the products with 16 bits or more, 24 where the
    result is float32 (two or three terms of 8 bits, each off by at most 2^-8 of what it stands for), and is rounded once at the end.
    Terms below 2^-126 may count as 0, as in layer_reference.dense_gradients; so may the last of two, where the value is below 2^-118."""
    dz_off = dz_off + 4 * 2.0 ** -126

    def through(a, b, off, dtype, depth):
        terms = 2.0 ** -24 if dtype == F32 else 2.0 ** -16
        size = a.abs() @ b.abs()
        return a @ b, off @ b.abs() + (terms + 3 * ref.E * (depth + 300)) * size
    gx, bx = through(dz, kg.values.t().contiguous(), dz_off, x_dtype, dz.shape[1])
    gk, bk = through(dz.t().contiguous(), xg.values, dz_off.t().contiguous(), k_dtype, dz.shape[0])
    gk, bk = gk.t() * kg.inside, bk.t() * kg.inside
    gx, bx = gx * xg.inside, bx * xg.inside
    return (gx, ref.rounded(gx, bx, x_dtype)), (gk, ref.rounded(gk, bk, k_dtype))


TYPES = [(BF16, BF16), (F32, BF16), (BF16, F32), (F16, BF16), (BF16, F16), (F16, F16), (F32, F32)]


@pytest.mark.parametrize("size", [(3, 5, 2), (45, 130, 127), (515, 333, 70), (1000, 300, 260)], ids=str)
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("x_dtype,k_dtype", TYPES, ids=str)
def test_products_of_gradients(pkg, noisy, size, activation, x_dtype, k_dtype):
    rows, depth, columns = size
    x, k = make((rows, depth), 1, x_dtype), make((depth, columns), 2, k_dtype)
    pre, gy = make((rows, columns), 3, x_dtype, 2.0), make((rows, columns), 4, x_dtype)
    g = pkg.FakeApproxDense(noisy, activation).gradients(gy, x, k, pre if activation else None)
    dz, off = gy.double(), torch.zeros((rows, columns), dtype=torch.float64, device=DEV)
    if activation:
        dz = dz * ref.slope(pre, activation)
        # a slope is a few operations of float32, whose exponentials' arguments z^2 / 2 or z are rounded
        off = gy.double().abs() * ref.E * (16 + 4 * pre.double().abs() + 4 * pre.double() ** 2)
    for name, got, (want, bound) in zip(("inputs", "kernel"), g, products(dz, off, ref.Grid(pkg, x), ref.Grid(pkg, k), x_dtype, k_dtype)):
        ref.check(got, want, bound, name)


@pytest.mark.parametrize("size", [(5, 64, 1000), (129, 64, 5003), (300, 48, 16390)], ids=str)
@pytest.mark.parametrize("x_dtype,k_dtype", [(BF16, BF16), (F32, BF16), (F16, F16)], ids=str)
def test_products_of_the_loss(pkg, noisy, size, x_dtype, k_dtype):
    rows, depth, vocabulary = size
    x, k = make((rows, depth), 1, x_dtype), make((depth, vocabulary), 2, k_dtype, depth ** -0.5)
    t = torch.arange(rows, device=DEV) * 7 % vocabulary
    _, g = pkg.FakeApproxCrossEntropy(noisy).loss_and_gradients(x, k, t)
    xg, kg = ref.Grid(pkg, x), ref.Grid(pkg, k)
    z, z_off = ref.product(pkg.synth.table_noisy(3), xg, kg)
    _, _, p, p_off = ref.loss(z, z_off, t, -100)
    dz = p.clone()
    dz[torch.arange(rows, device=DEV), t] -= 1
    dz, off = dz / rows, (p * p_off + 8 * ref.E * (p + dz.abs())) / rows
    for name, got, (want, bound) in zip(("inputs", "kernel"), g, products(dz, off, xg, kg, x_dtype, k_dtype)):
        ref.check(got, want, bound, name)


@pytest.mark.parametrize("common", [0.0, 1000.0, -131072.0])
@pytest.mark.parametrize("rows,vocabulary", [(3, 301), (45, 301), (45, 5003), (600, 5003)], ids=str)
def test_what_all_logits_have_in_common(pkg, noisy, rows, vocabulary, common):
    """Logits of x = 0 are the bias, exact here: multiples of 1/64 below 2^18.  The bound does not grow with their common part."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(vocabulary)
    part = torch.randint(-512, 513, (vocabulary,), device=DEV, generator=gen).double() / 64
    part[5] = 24.0                                  # rows of that target are sure of it
    bias = (part + common).float()
    assert torch.equal(bias.double(), part + common)
    x, k = torch.zeros((rows, 8), device=DEV), make((8, vocabulary), 2)
    t = torch.where(torch.arange(rows, device=DEV) % 2 == 0, 5, torch.arange(rows, device=DEV) * 11 % vocabulary)
    loss, g = pkg.FakeApproxCrossEntropy(noisy).loss_and_gradients(x, k, t, bias, "none")
    # a sum of exponentials in chunks, and those of differences up to 32, which are exact; then a log, and one sum
    log_sum = torch.log(torch.exp(part - 24.0).sum())
    want = (24.0 - part[t]) + log_sum
    off = torch.full_like(want, float(ref.E * (vocabulary / 64 + 256 + 4 * 32)))
    ref.check(loss, want, ref.rounded(want, off, F32), "loss")
    p = torch.exp(part - 24.0 - log_sum).expand(rows, -1)
    p_off = float(off[0]) + ref.E * (16 + 4 * (part - 24.0).abs())
    dz, dz_off = p.clone(), p * p_off
    dz[torch.arange(rows, device=DEV), t] -= 1
    dz_off = dz_off + 2 * ref.E * (p + dz.abs())
    sums, off = dz.sum(0), dz_off.sum(0) + (rows + 8) * ref.E * dz.abs().sum(0)
    ref.check(g.bias, sums, ref.rounded(sums, off, F32), "bias")
    (gx, gx_off), _ = products(dz, dz_off, ref.Grid(pkg, x), ref.Grid(pkg, k), F32, F32)
    ref.check(g.inputs, gx, gx_off, "inputs")


@pytest.mark.parametrize("rows", [1, 3, 45])
@pytest.mark.parametrize("activation", ["gelu", "gelu_tanh", "silu"])
def test_activations_over_their_tails(pkg, noisy, rows, activation):
    """What goes in is the bias, exact, as x is 0.  Bounds are relative to the result, however small: half steps of a few operations,
    and of an exponential's argument, once for each operation that made it: 4 for z^2 / 2, 8 for the cubic, 4 for z.  Beyond exp(87) a
    logistic function may be 0, off by 2^-125, and so may what an exponential below 2^-126 is multiplied by."""
    z = torch.linspace(-12.0, 12.0, 4803, device=DEV)
    layer = pkg.FakeApproxDense(noisy, activation)
    x, k = torch.zeros((rows, 8), device=DEV), make((8, z.numel()), 2)
    y, pre = layer.call_and_keep(x, k, z)
    assert torch.equal(pre, z.expand(rows, -1))
    d = z.double().requires_grad_()
    # (1 + tanh u) / 2 is the logistic function of 2 u; as it stands in layer_reference it is 1e-16 off, which is all there is below -8
    fn = (lambda v: v * torch.sigmoid(1.5957691216057308 * (v + 0.044715 * v ** 3))) if activation == "gelu_tanh" else \
        ref.ACTIVATIONS[activation]
    want = fn(d)
    slope = torch.autograd.grad(want.sum(), d)[0]
    want, d = want.detach(), d.detach()
    size = {"gelu": 3 * d * d, "gelu_tanh": 8 * 1.6 * (d + 0.044715 * d ** 3).abs(), "silu": 4 * d.abs()}[activation]
    bound = ref.E * (24 + size) * want.abs() + 2.0 ** -125 * d.abs()
    for row in y:
        ref.check(row, want, ref.rounded(want, bound, F32))
    # the slope, of one row: f + z f', either of which may be the larger
    g = layer.gradients(torch.ones_like(y[:1]), x[:1], k, pre[:1], want=("bias",)).bias
    terms = (want / d).abs() + (slope - want / d).abs()
    terms[d == 0] = 0.5
    ref.check(g, slope, ref.rounded(slope, ref.E * (32 + 2 * size) * terms + 2.0 ** -125 * (1 + d.abs() ** 3), F32), "slope")
