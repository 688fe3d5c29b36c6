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
