"""Transformer layers in approximate arithmetic, as measurable cases.

Every 8x8-bit product of a dense layer is a lookup T[a][b] in a 256x256 truth table, as in the framework's convolutions: both
operands are quantized to the 8-bit grid of their own (smallest, largest) value, a = code of the input, b = code of the kernel,

    product[m][n] = s_in * s_k * sum over k of (T[a][b] - z_k * a - z_in * b + z_in * z_k)

with scales s and zero points z.  A case is a plain dict.  "kind" says which operator it goes through:

  dense       residual + activation(product + bias); "packed": the kernel was laid out once, as a server keeps it
  dense_grad  its gradients for the input, the kernel and the bias: straight through the grid, where a value lies inside it
  loss        softmax cross entropy over a vocabulary whose logits are product + bias, and are not kept
  loss_grad   the loss and its gradients in one call
  norm        h = x + scale * gate * norm(block), y = norm(h): the norms before and after a block with its gate and scale
  norm_grad   its gradients for everything that went in

The grid is defined in float32, operation by operation, as the framework's fake quantization is.  Sizes are generic.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
IGNORE = -100

MAX_LOOKUPS = 2048 * 768 * 32000       # of a drawn case: the largest listed one
MAX_GRAD_WORK = 4096 * 1024 * 4096
MAX_NORM_VALUES = 16384 * 2048


def _dense(name, rows, depth, columns, dtype, activation=None, bias=True, residual=False, packed=False, kernel="same"):
    return {"name": name, "kind": "dense", "rows": rows, "depth": depth, "columns": columns, "dtype": dtype,
            "kernel_dtype": dtype if kernel == "same" else kernel, "activation": activation, "bias": bias,
            "residual": residual, "packed": packed}


def _dense_grad(name, rows, depth, columns, dtype, activation=None, kernel="same"):
    return {"name": name, "kind": "dense_grad", "rows": rows, "depth": depth, "columns": columns, "dtype": dtype,
            "kernel_dtype": dtype if kernel == "same" else kernel, "activation": activation}


def _loss(name, kind, rows, depth, columns, dtype, bias=False, reduction="mean"):
    return {"name": name, "kind": kind, "rows": rows, "depth": depth, "columns": columns, "dtype": dtype, "bias": bias,
            "reduction": reduction}


def _norm(name, kind, rows, width, dtype, norm="rms", post=False, gate_groups=0, scale=False, bias=False):
    return {"name": name, "kind": kind, "rows": rows, "width": width, "dtype": dtype, "norm": norm, "post": post,
            "gate_groups": gate_groups, "scale": scale, "bias": bias}


def listed():
    return [
        # one token of a server: latency, the kernel's bytes at most
        _dense("dense_token", 1, 1024, 4096, "bfloat16", bias=True, residual=True, packed=True),
        # a few requests' tokens together through a wide layer
        _dense("dense_tokens_8", 8, 4096, 4096, "bfloat16", activation="silu", bias=False, packed=True),
        # a short prompt, every size odd, float32 as in the convolutions
        _dense("dense_prompt_odd", 387, 1001, 1531, "float32", activation="gelu", residual=True),
        # a layer of a batch of long prompts, or of a training step forwards
        _dense("dense_prompt", 4096, 1024, 4096, "bfloat16", activation="gelu", kernel="float32"),
        # the same layer backwards
        _dense_grad("dense_grad", 4096, 1024, 4096, "bfloat16", activation="gelu"),
        # a small one in float32, odd sizes
        _dense_grad("dense_grad_odd", 515, 333, 1025, "float32", activation="relu"),
        # evaluation of a small model, per row
        _loss("loss_odd", "loss", 129, 512, 5003, "float32", bias=True, reduction="none"),
        # evaluation over an ordinary vocabulary
        _loss("loss_large", "loss", 2048, 768, 32000, "bfloat16"),
        # a training step's loss with its gradients
        _loss("loss_grad", "loss_grad", 1024, 512, 32000, "bfloat16"),
        # one token on its way between two blocks: latency
        _norm("norm_token", "norm", 1, 4096, "bfloat16", post=True),
        # odd width, LayerNorm, a gate for each of a batch's images and a scale for each channel
        _norm("norm_layer_odd", "norm", 6000, 1283, "float16", norm="layer", gate_groups=60, scale=True, bias=True),
        # a training step's norms backwards
        _norm("norm_grad", "norm_grad", 16384, 2048, "bfloat16", post=True, scale=True, gate_groups=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Most sizes are multiples of 64 or 8 as in real models, the rest anything."""
    n = _log_int(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    return max(lo, min(hi, n // step * step)) if n >= step else n


def draw(rng):
    kind = rng.choice(("dense", "dense", "dense_grad", "loss", "loss_grad", "norm", "norm_grad"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    if kind == "dense":
        packed = rng.random() < 0.5
        while True:
            c = _dense(None, _log_int(rng, 1, 64) if packed else _log_int(rng, 1, 8192), _size(rng, 16, 8192),
                       _size(rng, 16, 8192), dtype, rng.choice((None, "relu", "gelu", "silu")), rng.random() < 0.5,
                       rng.random() < 0.5, packed, rng.choice(("same", "float32")))
            if c["rows"] * c["depth"] * c["columns"] <= MAX_LOOKUPS / 2:
                break
    elif kind == "dense_grad":
        while True:
            c = _dense_grad(None, _log_int(rng, 1, 8192), _size(rng, 16, 4096), _size(rng, 16, 4096), dtype,
                            rng.choice((None, "relu", "gelu", "silu")))
            if c["rows"] * c["depth"] * c["columns"] <= MAX_GRAD_WORK:
                break
    elif kind in ("loss", "loss_grad"):
        most = MAX_LOOKUPS if kind == "loss" else MAX_LOOKUPS / 3
        while True:
            c = _loss(None, kind, _log_int(rng, 1, 4096), _size(rng, 32, 2048), _size(rng, 1000, 64000), dtype,
                      rng.random() < 0.5, rng.choice(("none", "sum", "mean")))
            if c["rows"] * c["depth"] * c["columns"] <= most:
                break
    else:
        while True:
            rows, groups = _log_int(rng, 1, 32768), rng.choice((0, 0, 1, -1))
            c = _norm(None, kind, rows, _size(rng, 16, 16384), dtype, rng.choice(("rms", "layer")), rng.random() < 0.5,
                      rows if groups < 0 else groups, rng.random() < 0.5, rng.random() < 0.5)
            if rows * c["width"] <= MAX_NORM_VALUES:
                break
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(shape, std=1.0, mean=0.0, dt=dtype):
        return torch.randn(shape, generator=gen, device=DEVICE).mul_(std).add_(mean).to(dt)

    s = {"case": case}
    if case["kind"] in ("norm", "norm_grad"):
        m, d = case["rows"], case["width"]
        s["x"], s["block"] = normal((m, d)), normal((m, d), 0.5, 0.1)
        s["weight"] = normal((d,), 0.1, 1.0)
        s["bias"] = normal((d,), 0.1) if case["bias"] else None
        s["post_weight"] = normal((d,), 0.1, 1.0) if case["post"] else None
        s["scale"] = normal((d,), 0.1, 0.3) if case["scale"] else None
        s["gate"] = normal((case["gate_groups"], d), 0.5, 0.5) if case["gate_groups"] else None
        if case["kind"] == "norm_grad":
            s["h"] = _plain_norm_forward(s, case)[0]
            s["grad_h"], s["grad_y"] = normal((m, d), 0.01), normal((m, d), 0.01)
        return s
    m, k, n = case["rows"], case["depth"], case["columns"]
    # a multiplier with a relative error of 2 %, as the synthetic tables of the framework's own cases
    a = torch.arange(256, device=DEVICE, dtype=torch.float64)
    products = a[:, None] * a[None, :]
    noise = torch.randn((256, 256), generator=gen, device=DEVICE, dtype=torch.float64)
    s["products"] = (products + torch.round(noise * 0.02 * products)).clamp_(0, 65535).to(torch.int32).reshape(-1)
    s["x"] = normal((m, k))
    kernel_dtype = DTYPES[case.get("kernel_dtype", case["dtype"])]
    s["kernel"] = normal((k, n), 1.0 / math.sqrt(k), dt=kernel_dtype)
    s["bias"] = normal((n,), 0.1, dt=kernel_dtype) if case.get("bias") else None
    if case["kind"] == "dense":
        s["residual"] = normal((m, n)) if case["residual"] else None
    elif case["kind"] == "dense_grad":
        s["pre"] = normal((m, n)) if case["activation"] else None
        s["grad"] = normal((m, n), 0.01)
    else:
        targets = torch.randint(0, n, (m,), generator=gen, device=DEVICE)
        ignored = torch.rand((m,), generator=gen, device=DEVICE) < 0.1
        s["targets"] = torch.where(ignored, torch.full_like(targets, IGNORE), targets)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import importlib
        pkg = importlib.import_module("tf-approximate_amd")
        if case["kind"] in ("norm", "norm_grad"):
            s["norm"] = pkg.ResidualNorm(case["norm"], 1e-6)
            return s
        s["table"] = pkg.TruthTable(s["products"].cpu().numpy().astype(np.uint16), 8)
        if case["kind"] in ("dense", "dense_grad"):
            s["layer"] = pkg.FakeApproxDense(s["table"], case["activation"])
            if case.get("packed"):
                s["packed"] = s["layer"].pack(s["kernel"])
        else:
            s["loss"] = pkg.FakeApproxCrossEntropy(s["table"], ignore_index=IGNORE)
    elif case.get("packed"):
        s["packed"] = _grid(s["kernel"])
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(s):
    return _RUN[s["case"]["kind"]](s, s["case"])


def _run_dense(s, c):
    if own:
        return s["layer"](s["x"], s["packed"] if c["packed"] else s["kernel"], s["bias"], s["residual"])
    z = _plain_product(s["products"], _grid(s["x"]), s["packed"] if c["packed"] else _grid(s["kernel"]))
    if s["bias"] is not None:
        z = z + s["bias"].float()
    z = _activation(z, c["activation"])
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(s["x"].dtype)


def _run_dense_grad(s, c):
    if own:
        g = s["layer"].gradients(s["grad"], s["x"], s["kernel"], s["pre"])
        return {"inputs": g.inputs, "kernel": g.kernel, "bias": g.bias}
    dz = s["grad"].float()
    if s["pre"] is not None:
        dz = dz * _slope(s["pre"].float(), c["activation"])
    dx, dk = _plain_product_grad(dz, s["x"], s["kernel"])
    return {"inputs": dx, "kernel": dk, "bias": dz.sum(0).to(s["kernel"].dtype)}


def _run_loss(s, c):
    if own:
        return s["loss"](s["x"], s["kernel"], s["targets"], s["bias"], c["reduction"])
    return _plain_loss(s, c)[0]


def _run_loss_grad(s, c):
    if own:
        loss, g = s["loss"].loss_and_gradients(s["x"], s["kernel"], s["targets"], s["bias"], c["reduction"])
        return {"loss": loss, "inputs": g.inputs, "kernel": g.kernel, "bias": g.bias}
    loss, p, counted, share = _plain_loss(s, c)
    rows = torch.arange(p.shape[0], device=p.device)
    p[rows, s["targets"].clamp(min=0)] -= 1.0
    p *= (counted.float() * share)[:, None]
    dx, dk = _plain_product_grad(p, s["x"], s["kernel"])
    return {"loss": loss, "inputs": dx, "kernel": dk, "bias": p.sum(0).to(s["kernel"].dtype) if c["bias"] else None}


def _run_norm(s, c):
    if own:
        return s["norm"](s["x"], s["block"], s["weight"], s["bias"], s["gate"], s["scale"], s["post_weight"])
    return _plain_norm_forward(s, c)


def _run_norm_grad(s, c):
    if own:
        g = s["norm"].gradients(s["grad_h"], s["grad_y"], s["h"], s["block"], s["weight"], s["bias"], s["gate"], s["scale"],
                                s["post_weight"])
        return {"x": g.x, "block": g.block, "weight": g.weight, "bias": g.bias, "gate": g.gate, "scale": g.scale,
                "post_weight": g.post_weight}
    dtype, m, d = s["x"].dtype, c["rows"], c["width"]
    dh, dw, db = _plain_norm_backward(s["grad_y"].float(), s["h"].float(), s["weight"].float(), c["norm"])
    dh = dh + s["grad_h"].float()
    block = s["block"].float()
    u = _plain_norm(block, s["post_weight"].float(), None, c["norm"]) if c["post"] else block
    gate = _rows_of_gate(s["gate"], m)
    factor = 1.0 if s["scale"] is None else s["scale"].float()
    factor = factor if gate is None else factor * gate
    du = dh * factor
    dgate = dscale = dpost = None
    if gate is not None:
        dgate = dh * u if s["scale"] is None else dh * u * s["scale"].float()
        dgate = dgate.reshape(c["gate_groups"], -1, d).sum(1).to(dtype)
    if s["scale"] is not None:
        dscale = (dh * u if gate is None else dh * u * gate).sum(0).to(dtype)
    if c["post"]:
        du, dpost, _ = _plain_norm_backward(du, block, s["post_weight"].float(), c["norm"])
        dpost = dpost.to(dtype)
    return {"x": dh.to(dtype), "block": du.to(dtype), "weight": dw.to(dtype),
            "bias": db.to(dtype) if s["bias"] is not None else None, "gate": dgate, "scale": dscale, "post_weight": dpost}


_RUN = {"dense": _run_dense, "dense_grad": _run_dense_grad, "loss": _run_loss, "loss_grad": _run_loss_grad,
        "norm": _run_norm, "norm_grad": _run_norm_grad}


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _grid(v):
    """The 8-bit grid of a tensor's own range, and its codes: (codes, scale, zero point, values inside the grid), in float32."""
    v = v.float()
    lo, hi = torch.aminmax(v)
    steps = torch.full((), 255.0, device=v.device)
    scale = (hi - lo) / steps
    zero = torch.floor((0.0 - lo / scale).clamp(0.0, 255.0) + 0.5)
    low, high = (0.0 - zero) * scale, (steps - zero) * scale
    codes = torch.floor((torch.minimum(torch.maximum(v, low), high) - low) * (torch.ones_like(scale) / scale) + 0.5)
    return codes.clamp_(0.0, 255.0).to(torch.int32), scale, zero, (v >= low) & (v <= high)


def _plain_product(products, x, kernel):
    """sum of table entries, in pieces of the rows, with what the zero points take away; whole numbers up to the last step."""
    a, s_in, z_in, _ = x
    b, s_k, z_k, _ = kernel
    m, k = a.shape
    piece = max(1, (1 << 26) // (k * b.shape[1]))
    sums = torch.cat([products.index_select(0, (rows[:, :, None] * 256 + b[None]).reshape(-1))
                      .reshape(rows.shape[0], k, -1).sum(1) for rows in a.split(piece)])
    z_in, z_k = z_in.long(), z_k.long()
    sums = sums - z_k * a.sum(1)[:, None] - z_in * b.sum(0) + k * z_in * z_k
    return sums.double().mul_(s_in.double() * s_k.double()).float()


def _plain_product_grad(dz, x, kernel):
    a, s_in, z_in, x_inside = _grid(x)
    b, s_k, z_k, k_inside = _grid(kernel)
    dx = torch.matmul(dz, ((b - z_k) * s_k).t().contiguous()) * x_inside
    dk = torch.matmul(((a - z_in) * s_in).t().contiguous(), dz) * k_inside
    return dx.to(x.dtype), dk.to(kernel.dtype)


def _plain_loss(s, c):
    """(loss, softmax, which rows count, what each contributes)"""
    z = _plain_product(s["products"], _grid(s["x"]), _grid(s["kernel"]))
    if s["bias"] is not None:
        z = z + s["bias"].float()
    top = z.max(1).values
    e = (z - top[:, None]).exp_()
    total = e.sum(1)
    counted = s["targets"] != IGNORE
    at = z.gather(1, s["targets"].clamp(min=0)[:, None])[:, 0]
    rows = torch.where(counted, total.log() + top - at, torch.zeros_like(top))
    share = torch.ones((), device=z.device)
    if c["reduction"] == "mean":
        share = share / counted.sum().clamp(min=1)
    loss = rows if c["reduction"] == "none" else rows.sum() * share
    return loss, e.div_(total[:, None]), counted, share


def _activation(z, name):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0.0).float()
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    sig = 1.0 / (1.0 + torch.exp(-z))
    return sig * (1.0 + z * (1.0 - sig))


def _plain_norm(v, weight, bias, kind):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-6) * weight
    return y if bias is None else y + bias


def _rows_of_gate(gate, rows):
    return None if gate is None else gate.float().repeat_interleave(rows // gate.shape[0], 0)


def _plain_norm_forward(s, c):
    u = s["block"].float()
    if c["post"]:
        u = _plain_norm(u, s["post_weight"].float(), None, c["norm"])
    if s["gate"] is not None:
        u = u * _rows_of_gate(s["gate"], c["rows"])
    if s["scale"] is not None:
        u = u * s["scale"].float()
    h = (s["x"].float() + u).to(s["x"].dtype)
    y = _plain_norm(h.float(), s["weight"].float(), None if s["bias"] is None else s["bias"].float(), c["norm"])
    return h, y.to(s["x"].dtype)


def _plain_norm_backward(dy, v, weight, kind):
    """(gradient for v, for the weight, for the bias)"""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    r = torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-6)
    n = v * r
    g = dy * weight
    dv = g - n * (g * n).mean(1, keepdim=True)
    if kind == "layer":
        dv = dv - g.mean(1, keepdim=True)
    return dv * r, (dy * n).sum(0), dy.sum(0)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    b = BYTES[case["dtype"]]
    if case["kind"] in ("norm", "norm_grad"):
        m, d = case["rows"], case["width"]
        vectors = 1 + case["bias"] + case["post"] + case["scale"] + case["gate_groups"]
        if case["kind"] == "norm":   # x, block in; h, y out
            return {"bytes": b * (4 * m * d + vectors * d), "flops": 12 * m * d}
        return {"bytes": b * (6 * m * d + 2 * vectors * d), "flops": 30 * m * d}   # two gradients, h, block in; two out
    m, k, n = case["rows"], case["depth"], case["columns"]
    kb = BYTES[case.get("kernel_dtype", case["dtype"])]
    product = 2 * m * k * n
    if case["kind"] == "dense":
        kernel = k * n * (1 if case["packed"] else kb)
        return {"bytes": b * m * k + kernel + kb * n * case["bias"] + b * m * n * (1 + case["residual"]) + 131072,
                "flops": product}
    if case["kind"] == "dense_grad":
        pre = 1 if case["activation"] else 0
        return {"bytes": b * (2 * m * k + (1 + pre) * m * n) + kb * (2 * k * n + n), "flops": 2 * product}
    once = b * (m * k + k * n + n * case["bias"]) + 8 * m + 4 * m + 131072
    if case["kind"] == "loss":
        return {"bytes": once, "flops": product}
    return {"bytes": once + b * (m * k + k * n), "flops": 3 * product}


# ---- the definitions in 64 bits, apart from the above ------------------------------------------------------------------

def _codes64(t):
    """Codes minus zero point, codes, zero point, scale and the mask of values inside the grid.  What the grid is, is defined in
    float32, one rounding an operation; numpy does them."""
    v = t.float().cpu().numpy()
    f = np.float32
    lo, hi = f(v.min()), f(v.max())
    scale = f(f(hi - lo) / f(255.0))
    at = f(f(0.0) - f(lo / scale))
    zero = 0 if at < 0 else 255 if at > 255 else int(math.floor(float(at) + 0.5))
    low, high = f(f(0 - zero) * scale), f(f(255 - zero) * scale)
    inverse = f(f(1.0) / scale)
    q = np.floor((np.clip(v, low, high) - low).astype(f) * inverse + f(0.5)).astype(np.int64).clip(0, 255)
    inside = torch.from_numpy(((v >= low) & (v <= high))).to(DEVICE).double()
    q = torch.from_numpy(q).to(DEVICE)
    return (q - zero).double(), q, zero, float(scale), inside


def _logits64(s):
    xc, a, za, sa, x_in = _codes64(s["x"])
    kc, b, zb, sb, k_in = _codes64(s["kernel"])
    # entry minus the two zero points' part, one filter element after the other
    codes = torch.arange(256, device=DEVICE, dtype=torch.float64)
    entry = s["products"].double().view(256, 256) - zb * codes[:, None] - za * codes[None, :] + za * zb
    total = torch.zeros((a.shape[0], b.shape[1]), dtype=torch.float64, device=DEVICE)
    for k in range(a.shape[1]):
        total += entry[:, b[k]][a[:, k]]
    z = total * (sa * sb)
    if s["bias"] is not None:
        z += s["bias"].double()
    return z, xc * sa, kc * sb, x_in, k_in


def _norm64(v, w, b, kind, eps=1e-6):
    mean = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    var = ((v - mean) ** 2).mean(1, keepdim=True)
    y = (v - mean) / torch.sqrt(var + eps) * w
    return y + b if b is not None else y


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        d = {k: (v.double() if torch.is_tensor(v) else v) for k, v in s.items()}
        each = case["rows"] // case["gate_groups"] if case["gate_groups"] else 1

        def between(block, post, gate, scale):
            u = block if post is None else _norm64(block, post, None, case["norm"])
            if gate is not None:
                u = u * gate[torch.arange(case["rows"], device=DEVICE) // each]
            return u if scale is None else u * scale

        if kind == "norm":
            h = d["x"] + between(d["block"], d["post_weight"], d["gate"], d["scale"])
            return h, _norm64(h, d["weight"], d["bias"], case["norm"])
        leaves = {k: d[k].requires_grad_() for k in ("block", "weight", "bias", "gate", "scale", "post_weight", "h")
                  if d[k] is not None}
        with torch.enable_grad():
            y = _norm64(d["h"], d["weight"], d["bias"], case["norm"])
            g1 = torch.autograd.grad((y * d["grad_y"]).sum(), [leaves[k] for k in ("h", "weight", "bias") if k in leaves])
            dh = g1[0] + d["grad_h"]
            rest = [k for k in ("block", "gate", "scale", "post_weight") if k in leaves]
            u = between(d["block"], d["post_weight"], d["gate"], d["scale"])
            g2 = dict(zip(rest, torch.autograd.grad((u * dh.detach()).sum(), [leaves[k] for k in rest])))
        return {"x": dh.detach(), "block": g2["block"], "weight": g1[1], "bias": g1[2] if len(g1) > 2 else None,
                "gate": g2.get("gate"), "scale": g2.get("scale"), "post_weight": g2.get("post_weight")}
    if kind == "dense_grad":
        dz = s["grad"].double()
        if s["pre"] is not None:
            pre = s["pre"].double().requires_grad_()
            with torch.enable_grad():
                f = {"relu": lambda v: v * (v > 0), "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2.0)),
                     "silu": lambda v: v * torch.sigmoid(v)}[case["activation"]]
                dz, = torch.autograd.grad((f(pre) * dz).sum(), [pre])
        xc, _, _, sa, x_in = _codes64(s["x"])
        kc, _, _, sb, k_in = _codes64(s["kernel"])
        return {"inputs": (dz @ kc.t().contiguous()) * sb * x_in, "kernel": (xc.t().contiguous() @ dz) * sa * k_in,
                "bias": dz.sum(0)}
    z, xv, kv, x_in, k_in = _logits64(s)
    if kind == "dense":
        act = case["activation"]
        if act == "relu":
            z = torch.where(z > 0, z, torch.zeros_like(z))
        elif act == "gelu":
            z = z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
        elif act == "silu":
            z = z * torch.sigmoid(z)
        return z + s["residual"].double() if s["residual"] is not None else z
    t = s["targets"]
    counted = (t != IGNORE).double()
    log_p = z - torch.logsumexp(z, 1, keepdim=True)
    rows = -log_p[torch.arange(t.shape[0], device=DEVICE), t.clamp(min=0)] * counted
    weight = counted / max(1.0, float(counted.sum())) if case["reduction"] == "mean" else counted
    loss = rows if case["reduction"] == "none" else (rows * weight).sum()
    if kind == "loss":
        return loss
    dz = log_p.exp()
    dz[torch.arange(t.shape[0], device=DEVICE), t.clamp(min=0)] -= 1.0
    dz *= weight[:, None]
    return {"loss": loss, "inputs": (dz @ kv.t().contiguous()) * x_in, "kernel": (xv.t().contiguous() @ dz) * k_in,
            "bias": dz.sum(0) if case["bias"] else None}
