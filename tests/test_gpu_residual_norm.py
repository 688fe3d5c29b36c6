"""ResidualNorm against its definition in 64 bits, and the layers together as a model has them."""
import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"
EPS = 1e-5


def make(shape, seed, dtype=F32, std=1.0, mean=0.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=gen) * std + mean).to(dtype)


class Case:
    def __init__(self, rows, width, dtype, vector_dtype, kind, groups, what):
        self.kind, self.rows, self.width, self.groups = kind, rows, width, groups
        self.x, self.block = make((rows, width), 1, dtype), make((rows, width), 2, dtype, 0.7, 0.4)
        self.weight = make((width,), 3, vector_dtype, 0.2, 1.0)
        self.bias = make((width,), 4, vector_dtype) if "bias" in what else None
        self.scale = make((width,), 5, vector_dtype, 0.3, 0.5) if "scale" in what else None
        self.post = make((width,), 6, vector_dtype, 0.2, 1.0) if "post" in what else None
        self.gate = make((groups, width), 7, dtype) if groups else None

    def args(self):
        return self.block, self.weight, self.bias, self.gate, self.scale, self.post

    def gate_rows(self):
        return self.gate.double().repeat_interleave(self.rows // self.groups, 0)

    def u(self):
        """(u, bound)"""
        b = self.block.double()
        if self.post is None:
            return b, torch.zeros_like(b)
        n, _, off = ref.normed(b, self.kind, EPS)
        w = self.post.double()
        return n * w, (off + 2 * ref.E * n.abs()) * w.abs()

    def h(self):
        u, off = self.u()
        for f in ((self.gate_rows() if self.groups else None), (None if self.scale is None else self.scale.double())):
            if f is not None:
                u, off = u * f, (off + 2 * ref.E * u.abs()) * f.abs()
        h = self.x.double() + u
        return h, off + 2 * ref.E * h.abs()

    def y(self, h):
        n, _, off = ref.normed(h.double(), self.kind, EPS)
        w = self.weight.double()
        y, off = n * w, (off + 2 * ref.E * n.abs()) * w.abs()
        if self.bias is not None:
            y = y + self.bias.double()
            off = off + 2 * ref.E * y.abs()
        return y, off


ALL = ("bias", "scale", "post")
CASES = [
    # width around lanes, vectors, workgroups; off the fours; the widest
    (1, 1, 0, ()), (3, 2, 3, ALL), (5, 4, 1, ("post",)), (7, 63, 7, ("scale",)), (64, 64, 8, ALL), (10, 255, 5, ("bias",)),
    (33, 256, 0, ALL), (9, 1283, 3, ALL), (40, 2048, 2, ("post", "bias")), (6, 2052, 1, ALL), (5, 4096, 5, ALL), (4, 4099, 2, ALL),
    (3, 8192, 1, ("scale",)), (3, 8193, 3, ALL), (2, 16384, 1, ALL), (2, 32768, 2, ALL), (2, 32767, 1, ALL),
    # more rows than workgroups, groups of whole runs and runs of whole groups
    (1200, 40, 2, ALL), (5000, 24, 1000, ALL), (4097, 17, 0, ALL), (3000, 36, 3000, ("scale",)),
    (1600, 4100, 4, ALL), (1600, 4101, 1600, ("post",)), (1100, 8197, 550, ALL), (1030, 8196, 0, ("scale", "bias")),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype,vector_dtype", [(F32, F32), (BF16, F32), (F16, BF16)], ids=str)
def test_forward_and_gradients(pkg, case, kind, dtype, vector_dtype):
    print("case", case, kind, dtype, vector_dtype, flush=True)
    rows, width, groups, what = case
    c = Case(rows, width, dtype, vector_dtype, kind, groups, what)
    norm = pkg.ResidualNorm(kind, EPS)
    h, y, seen = norm.call_in_turn(c.x, *c.args())
    want, off = c.h()
    ref.check(h, want, ref.rounded(want, off, dtype), "h")
    want, off = c.y(h)
    ref.check(y, want, ref.rounded(want, off, dtype), "y")
    pairs = seen.view(-1, 2)
    lo, hi = torch.aminmax(y)
    assert float(pairs[:, 0].min()) == float(lo) and float(pairs[:, 1].max()) == float(hi)
    h2, y2 = norm(c.x, *c.args())
    assert torch.equal(h, h2) and torch.equal(y, y2)

    gh, gy = make(h.shape, 8, dtype), make(h.shape, 9, dtype)
    g = norm.gradients(gh, gy, h, *c.args())
    hd, E = h.double(), ref.E
    w = c.weight.double()
    dn = gy.double() * w
    dh, dh_off = ref.norm_backward(dn, 2 * E * dn.abs(), hd, kind, EPS)
    dh, dh_off = dh + gh.double(), dh_off + 2 * E * (dh + gh.double()).abs()
    ref.check(g.x, dh, ref.rounded(dh, dh_off, dtype), "x")
    n, _, n_off = ref.normed(hd, kind, EPS)

    def sums(v, off, shape=None):   # over rows: a run after the other, in any order at most `rows` additions
        v, off, size = (t if shape is None else t.reshape(shape) for t in (v, off, v.abs()))
        axis = 0 if shape is None else 1
        return v.sum(axis), off.sum(axis) + (v.shape[axis] + 8) * E * size.sum(axis)

    def check(got, v, off, name, shape=None):
        s, o = sums(v, off, shape)
        ref.check(got, s, ref.rounded(s, o, got.dtype), name)

    check(g.weight, gy.double() * n, gy.double().abs() * (n_off + 2 * E * n.abs()), "weight")
    if c.bias is not None:
        check(g.bias, gy.double(), torch.zeros_like(dh), "bias")
    u, u_off = c.u()
    hu, hu_off = dh * u, dh_off * u.abs() + dh.abs() * (u_off + 3 * E * u.abs())
    gate = c.gate_rows() if groups else torch.ones_like(dh)
    scale = torch.ones(width, dtype=torch.float64, device=DEV) if c.scale is None else c.scale.double()
    if c.scale is not None:
        check(g.scale, hu * gate, (hu_off + 2 * E * hu.abs()) * gate.abs(), "scale")
    if groups:
        check(g.gate, hu * scale, (hu_off + 2 * E * hu.abs()) * scale.abs(), "gate", (groups, rows // groups, width))
    du, du_off = dh * scale * gate, (dh_off + 4 * E * dh.abs()) * (scale * gate).abs()
    if c.post is not None:
        bn, _, bn_off = ref.normed(c.block.double(), kind, EPS)
        check(g.post_weight, du * bn, du_off * bn.abs() + du.abs() * (bn_off + 2 * E * bn.abs()), "post_weight")
        p = c.post.double()
        du, du_off = ref.norm_backward(du * p, (du_off + 2 * E * du.abs()) * p.abs(), c.block.double(), kind, EPS)
    ref.check(g.block, du, ref.rounded(du, du_off, dtype), "block")
    assert [t is None for t in g] == [False] + [t is None for t in (c.block, c.weight, c.bias, c.gate, c.scale, c.post)]
    # either gradient alone
    zero = torch.zeros_like(gh)
    for a, b in ((gh, None), (None, gy)):
        part = norm.gradients(a, b, h, *c.args())
        whole = norm.gradients(zero if a is None else a, zero if b is None else b, h, *c.args())
        for v, t in zip(part, whole):
            assert v is None or torch.equal(v, t)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", [24, 31, 3000])
def test_without_a_block(pkg, kind, width):
    x, w, gy, gh = make((5, width), 1), make((width,), 2), make((5, width), 3), make((5, width), 4)
    norm = pkg.ResidualNorm(kind, EPS)
    h, y = norm(x, None, w)
    assert h is x
    n, _, off = ref.normed(x.double(), kind, EPS)
    want = n * w.double()
    ref.check(y, want, ref.rounded(want, (off + 2 * ref.E * n.abs()) * w.abs(), F32))
    g = norm.gradients(gh, gy, h, None, w)
    dn = gy.double() * w.double()
    dv, off = ref.norm_backward(dn, 2 * ref.E * dn.abs(), x.double(), kind, EPS)
    want = dv + gh.double()
    ref.check(g.x, want, ref.rounded(want, off + 2 * ref.E * want.abs(), F32))
    assert g.block is None and g.gate is None


def test_gradient_is_a_difference(pkg):
    """Of sum(wh h + wy y) by steps of x and block; the second derivative's part cancels, the third's is below h^2 of values
    around 1, the outputs' rounding counts over 2 h."""
    for kind in ("rms", "layer"):
        c = Case(4, 40, F32, F32, kind, 2, ALL)
        norm = pkg.ResidualNorm(kind, EPS)
        wh, wy = make((4, 40), 8), make((4, 40), 9)

        def total():
            h, y = norm(c.x, *c.args())
            return float((wh.double() * h.double() + wy.double() * y.double()).sum())

        h, _ = norm(c.x, *c.args())
        g = norm.gradients(wh, wy, h, *c.args())
        step = 2.0 ** -6
        for t, d in ((c.x, g.x), (c.block, g.block), (c.gate, g.gate), (c.scale, g.scale), (c.post, g.post_weight),
                     (c.weight, g.weight), (c.bias, g.bias)):
            flat, at = t.view(-1), t.numel() // 3
            kept = float(flat[at])
            flat[at] = kept + step
            up, moved_up = total(), float(flat[at])
            flat[at] = kept - step
            down, moved_down = total(), float(flat[at])
            flat[at] = kept
            noise = 16 * ref.E * float((wh.abs() * h.abs()).sum() + (wy.abs() * 3).sum()) / step
            assert abs((up - down) / (moved_up - moved_down) - float(d.view(-1)[at])) <= noise + 20 * step * step


def test_rows_of_zeros_and_infinities(pkg):
    for kind in ("rms", "layer"):
        c = Case(6, 52, F32, F32, kind, 0, ("post",))
        c.x[2] = 0
        c.block[2] = 0
        c.x[4, 7] = float("inf")
        norm = pkg.ResidualNorm(kind, EPS)
        h, y = norm(c.x, *c.args())
        assert not h[2].any() and not y[2].any()
        assert torch.isnan(y[4]).any() and torch.isfinite(y[[0, 1, 2, 3, 5]]).all()
        g = norm.gradients(torch.ones_like(h), torch.ones_like(h), h, *c.args())
        assert torch.isfinite(g.x[[0, 1, 2, 3, 5]]).all() and torch.isfinite(g.block[[0, 1, 2, 3, 5]]).all()


def test_alignment_and_strides(pkg):
    norm = pkg.ResidualNorm("rms", EPS)
    for dtype in (F32, BF16):
        c = Case(6, 64, dtype, F32, "rms", 3, ALL)
        want = norm(c.x, *c.args())
        wg = norm.gradients(c.x, c.block, want[0], *c.args())

        def moved(t):
            m = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
            return m.copy_(t)

        m = [moved(t) for t in (c.x,) + c.args()]
        got = norm(*m)
        mg = norm.gradients(m[0], m[1], moved(want[0]), *m[1:])
        for a, b in zip(got + tuple(mg), want + tuple(wg)):   # sums of a row in another order, then the type's rounding
            assert (a.double() - b.double()).abs().max() <= 3 * ref.half_step(dtype) * b.double().abs().max()
        apart = torch.zeros((6, 2, 64), dtype=dtype, device=DEV)
        apart[:, 1] = c.x
        assert torch.equal(norm(apart[:, 1], *c.args())[1], want[1])


def test_far_rows(pkg):
    """More than 2^31 elements: the last rows, against a call on those alone."""
    norm = pkg.ResidualNorm("rms", EPS)
    rows, width = 270000, 8192
    x, w = make((rows, width), 1, BF16), make((width,), 2, BF16, 0.1, 1.0)
    assert x.numel() > 2 ** 31
    _, y, seen = norm.call_in_turn(x, x, w)
    h, last = norm(x[-30:], x[-30:], w)
    assert torch.equal(y[-30:], last)
    g = norm.gradients(y, y, x, None, w)
    assert torch.equal(g.x[-30:], norm.gradients(y[-30:], y[-30:], x[-30:], None, w).x)
    pairs = seen.view(-1, 2)
    lo, hi = torch.aminmax(y)
    assert float(pairs[:, 0].min()) == float(lo) and float(pairs[:, 1].max()) == float(hi)


def test_gates_of_a_batch(pkg):
    norm = pkg.ResidualNorm("layer", EPS)
    x, b, w = make((3, 5, 32), 1), make((3, 5, 32), 2), make((32,), 3)
    gate = make((3, 1, 32), 4)
    h, y = norm(x, b, w, gate=gate)
    flat = norm(x.view(15, 32), b.view(15, 32), w, gate=gate.expand(3, 5, 32).reshape(15, 32))
    assert h.shape == x.shape and torch.equal(h.view(15, 32), flat[0]) and torch.equal(y.view(15, 32), flat[1])
    assert norm.gradients(h, y, h, b, w, gate=gate).gate.shape == (3, 1, 32)
    with pytest.raises(pkg.InvalidArgumentError):
        norm(x, b, w, gate=gate[:2])
    with pytest.raises(pkg.InvalidArgumentError):
        norm(x, None, w, gate=gate)
    with pytest.raises(pkg.InvalidArgumentError):
        norm(x, b.to(BF16), w)
    with pytest.raises(pkg.InvalidArgumentError):
        norm(x, b, w[:5])
    with pytest.raises(pkg.InvalidArgumentError):
        norm(x, b, w, scale=w.to(BF16))
    with pytest.raises(pkg.InvalidArgumentError):
        norm(x, b, w.cpu())
    with pytest.raises(pkg.UnimplementedError):
        norm(x.double(), b.double(), w)
    empty = norm(x[:0], b[:0], w)
    assert empty[0].shape == (0, 5, 32)
    g = norm.gradients(x[:0], x[:0], x[:0], b[:0], w, bias=w)
    assert not g.weight.any() and not g.bias.any() and g.x.shape == (0, 5, 32)


# ---- the layers together ----

class Block:
    """norm, dense with its activation, dense, norm with the residual sum, loss; and backwards."""

    def __init__(self, pkg, rows, width, hidden, vocabulary, dtype, seed=0):
        self.pkg = pkg
        self.table = pkg.synth.table_noisy(3)
        handle = pkg.ops.TruthTable(self.table)
        self.norm = pkg.ResidualNorm("rms", EPS)
        self.up, self.down = pkg.FakeApproxDense(handle, "gelu"), pkg.FakeApproxDense(handle)
        self.loss = pkg.FakeApproxCrossEntropy(handle)
        self.x = make((rows, width), seed + 1, dtype)
        self.w1, self.w2 = make((width,), seed + 2, F32, 0.1, 1.0), make((width,), seed + 3, F32, 0.1, 1.0)
        self.post = make((width,), seed + 4, F32, 0.1, 1.0)
        self.k1 = make((width, hidden), seed + 5, dtype, width ** -0.5)
        self.k2 = make((hidden, width), seed + 6, dtype, hidden ** -0.5)
        self.head = make((width, vocabulary), seed + 7, dtype, width ** -0.5)
        self.b1 = make((hidden,), seed + 8, dtype, 0.1)
        self.targets = torch.randint(0, vocabulary, (rows,), device=DEV)
        self.targets[::7] = -100

    def step(self, in_turn=True):
        s = {}
        _, s["y"], r1 = self.norm.call_in_turn(self.x, None, self.w1)
        s["a"], s["pre"] = self.up.call_and_keep(s["y"], self.k1, self.b1, input_range=r1 if in_turn else None)
        s["b"] = self.down(s["a"], self.k2)
        s["h"], s["z"], r2 = self.norm.call_in_turn(self.x, s["b"], self.w2, post_weight=self.post)
        s["loss"], gl = self.loss.loss_and_gradients(s["z"], self.head, self.targets, input_range=r2 if in_turn else None)
        gn = self.norm.gradients(None, gl.inputs, s["h"], s["b"], self.w2, post_weight=self.post)
        gd = self.down.gradients(gn.block, s["a"], self.k2)
        gu = self.up.gradients(gd.inputs, s["y"], self.k1, s["pre"], input_range=r1 if in_turn else None)
        gx = self.norm.gradients(gn.x, gu.inputs, self.x, None, self.w1)
        s.update(gz=gl.inputs, head=gl.kernel, gb=gn.block, gh=gn.x, w2=gn.weight, post=gn.post_weight, ga=gd.inputs, k2=gd.kernel,
                 gy=gu.inputs, k1=gu.kernel, b1=gu.bias, gx=gx.x, w1=gx.weight)
        return s


@pytest.mark.parametrize("rows,width,hidden,vocabulary,dtype", [(3, 40, 72, 1001, F32), (150, 64, 200, 3001, F32),
                                                                (90, 128, 256, 2000, BF16)], ids=str)
def test_together(pkg, rows, width, hidden, vocabulary, dtype):
    m = Block(pkg, rows, width, hidden, vocabulary, dtype)
    s = m.step()
    # ranges handed on change nothing
    for a, b in zip(s.values(), m.step(in_turn=False).values()):
        assert torch.equal(a, b)
    # each part's result against the definition, from the inputs it had
    G = lambda t: ref.Grid(pkg, t)  # noqa: E731
    want, z, off, z_off = ref.dense(m.table, G(s["y"]), G(m.k1), m.b1, None, "gelu")
    ref.check(s["a"], want, ref.rounded(want, off, dtype), "up")
    want, _, off, _ = ref.dense(m.table, G(s["a"]), G(m.k2))
    ref.check(s["b"], want, ref.rounded(want, off, dtype), "down")
    logits, off = ref.product(m.table, G(s["z"]), G(m.head))
    losses, bound, p, p_off = ref.loss(logits, off, m.targets, -100)
    count = int((m.targets != -100).sum())
    ref.check(s["loss"], losses.sum() / count, ref.rounded(losses.sum() / count, bound.sum() / count, F32), "loss")
    share = (m.targets != -100).double() / count
    dz = p.clone()
    dz[torch.arange(rows, device=DEV), m.targets.clamp(min=0)] -= 1
    dz, dz_off = dz * share[:, None], (p * p_off + 8 * ref.E * (p + dz.abs())) * share[:, None]
    (gz, gz_off), (gk, gk_off), _ = ref.dense_gradients(dz, dz_off, G(s["z"]), G(m.head), dtype, dtype)
    ref.check(s["gz"], gz, gz_off, "gz")
    ref.check(s["head"], gk, gk_off, "head")
    (ga, ga_off), (gk, gk_off), _ = ref.dense_gradients(s["gb"].double(), torch.zeros_like(s["gb"].double()), G(s["a"]), G(m.k2),
                                                        dtype, dtype)
    ref.check(s["ga"], ga, ga_off, "ga")
    ref.check(s["k2"], gk, gk_off, "k2")


def test_a_range_is_that_of_its_tensor_as_it_was(pkg):
    m = Block(pkg, 40, 64, 72, 100, F32)
    _, y, seen = m.norm.call_in_turn(m.x, None, m.w1)
    want = m.up(y, m.k1)
    assert torch.equal(m.up(y, m.k1, input_range=seen), want)
    other = 3 * y
    assert torch.equal(m.up(other, m.k1, input_range=seen), m.up(other, m.k1))
    y.mul_(2.0)                                       # written to since
    assert torch.equal(m.up(y, m.k1, input_range=seen), m.up(y, m.k1))
    with pytest.raises(pkg.InvalidArgumentError):
        m.up(y, m.k1, input_range=seen[:10])
    # a convolution's range, and a dense layer's input for a convolution
    conv = pkg.FakeApproxConv2D((1, 1), m.up.table, "VALID")
    _, y, seen = m.norm.call_in_turn(m.x.view(1, 5, 8, 64), None, m.w1)
    k = make((1, 1, 64, 16), 3)
    assert torch.equal(conv.call_in_turn(y, k, input_range=seen)[0], conv(y, k))


def test_together_in_a_graph(pkg):
    m = Block(pkg, 130, 64, 128, 2000, BF16)
    m.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = m.step()
    for trial in range(4):
        m.x.copy_(make(m.x.shape, 70 + trial, BF16))
        m.k1.add_(make(m.k1.shape, 80 + trial, BF16, 0.01))
        want = m.step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in s:
            assert torch.equal(s[name], want[name]), name


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_no_rows(pkg, kind):
    norm = pkg.ResidualNorm(kind, EPS)
    x, w, gate = make((0, 3, 32), 1), make((32,), 3), make((1, 32), 4)
    args = (x, w, w, gate, w, w)
    h, y, seen = norm.call_in_turn(x, *args)
    assert h.shape == x.shape and y.shape == x.shape and seen is None
    assert norm(x, x, w, gate=make((0, 32), 4), scale=w)[0].shape == x.shape
    g = norm.gradients(h, y, h, *args)
    assert g.x.shape == x.shape and g.block.shape == x.shape
    for sums in (g.weight, g.bias, g.scale, g.post_weight, g.gate):
        assert not sums.any()


@pytest.mark.parametrize("rows,width", [(1, 40), (2, 8192), (5, 300), (33, 64)])
def test_a_norm_s_range_for_a_layer(pkg, rows, width):
    """A layer that is handed its input's range, of few rows as of many, has the results of one that looks for it."""
    norm, layer = pkg.ResidualNorm("rms", EPS), pkg.FakeApproxDense(pkg.ops.TruthTable(pkg.synth.table_noisy(3)), "silu")
    x, b, w, k = make((rows, width), 1, BF16), make((rows, width), 2, BF16), make((width,), 3), make((width, 50), 4, BF16)
    h, y, seen = norm.call_in_turn(x, b, w)
    for kernel in (k, layer.pack(k)):
        assert torch.equal(layer(y, kernel, residual=None, input_range=seen), layer(y, kernel))
    out, pre = layer.call_and_keep(y, k)
    for a, c in zip(layer.gradients(out, y, k, pre, input_range=seen), layer.gradients(out, y, k, pre)):
        assert torch.equal(a, c)
