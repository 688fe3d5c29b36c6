"""Transformer layers in approximate arithmetic: what stands around FakeApproxConv2D's arithmetic in a model made of dense layers.

    FakeApproxDense          residual + activation(product + bias), the product through the truth table; its gradients
    FakeApproxCrossEntropy   softmax cross entropy over a vocabulary whose logits go through the table, and are not kept
    ResidualNorm             the norms before and after a block with its gate and scale; reports the range of what it makes

The reference has no table op but the convolution: its layer call (tf2/python/keras/layers/fake_approx_convolutional.py:223-261,
min / max of both operands, fake quantization, the op, bias, activation) is made here around matrix products.  As everywhere in
this package torch owns the memory and the stream, and all arithmetic happens in libaxconv_hip.so.  Calls take no part in
torch.autograd: gradients are calls of their own, and can be captured into a graph as forward passes can.  A forward call on a tensor
that requires a gradient is therefore refused while torch records (under torch.no_grad() it is not).  Every call has
scratch memory of its own from torch's allocator, so calls on several streams, and graphs, do not meet in it.
"""
import collections
import ctypes
import math
import weakref

import torch

from . import _lib
from .ops import InvalidArgumentError, UnimplementedError, TruthTable, _check, _launch, _stream, _version

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_NORMS = {"rms": 0, "layer": 1}

DenseGradients = collections.namedtuple("DenseGradients", "inputs kernel bias")
ResidualNormGradients = collections.namedtuple("ResidualNormGradients", "x block weight bias gate scale post_weight")


def _require(t, what, device=None, dtype=None, shape=None):
    """A contiguous tensor on the GPU, of a type the layers have."""
    if not torch.is_tensor(t) or not t.is_cuda:
        raise InvalidArgumentError("%s must be a tensor on the GPU" % what)
    if t.dtype not in _TYPES:
        raise UnimplementedError("%s: only float32, bfloat16 and float16" % what)
    if device is not None and t.device != device:
        raise InvalidArgumentError("%s is on another device than the input" % what)
    if dtype is not None and t.dtype != dtype:
        raise InvalidArgumentError("%s must be %s, as what it goes with" % (what, dtype))
    if shape is not None and t.shape != shape:
        raise InvalidArgumentError("%s must have the shape %s" % (what, tuple(shape)))
    return t if t.is_contiguous() else t.contiguous()


def _unrecorded(*tensors):
    """Torch would take the output for a constant, and what it comes from would silently have no gradient."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and getattr(t, "requires_grad", False):
                raise InvalidArgumentError("a gradient does not pass through this call: make it under torch.no_grad(), and take "
                                           "gradients() for what requires one")


def _pointer(t):
    return None if t is None else t.data_ptr()


def _scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _range_pointer(input_range, inputs):
    """Where the range that a call reported of `inputs` is; None if there is none, or it is that of another tensor, or of this one
    before it was written to."""
    if input_range is None:
        return None
    if not torch.is_tensor(input_range) or input_range.device != inputs.device:
        raise InvalidArgumentError("input_range must be a tensor on the input's GPU")
    if (input_range.dtype != torch.float32 or not input_range.is_contiguous() or
            input_range.numel() * 4 < _lib.RANGE_BYTES):
        raise InvalidArgumentError("input_range must be what a call in turn returned")
    of, version = getattr(input_range, "_range_of", (None, None))
    if version is None or of() is not inputs or _version(inputs) != version:
        return None
    return input_range.data_ptr()


class PackedKernel:
    """A kernel's codes, laid out once by FakeApproxDense.pack for many calls.  Later changes of the kernel do not reach it."""

    def __init__(self, data, depth, columns, dtype):
        self.data, self.depth, self.columns, self.dtype = data, depth, columns, dtype


def _dense_desc(inputs, depth, columns, kernel_dtype, bias, activation, minmax):
    if inputs.dim() < 1 or inputs.shape[-1] != depth:
        raise InvalidArgumentError("the input's last axis must be the kernel's depth, %d" % depth)
    lo, hi = minmax if minmax is not None else (0.0, 0.0)
    return _lib.DenseDesc(inputs.numel() // depth if depth else 0, depth, columns, _TYPES[inputs.dtype], _TYPES[kernel_dtype],
                          _lib.F32 if bias is None else _TYPES[bias.dtype], activation, minmax is not None, lo, hi)


def _kernel_of(kernel, device):
    kernel = _require(kernel, "kernel", device)
    if kernel.dim() != 2:
        raise InvalidArgumentError("kernel must be 2-dimensional, [depth, columns]")
    return kernel


def _minmax_of(input_minmax):
    if input_minmax is None:
        return None
    lo, hi = (float(v) for v in input_minmax)
    if not lo <= hi or lo in (float("inf"), float("-inf")) or hi in (float("inf"), float("-inf")):
        raise InvalidArgumentError("input_minmax must be a finite (smallest, largest)")
    return lo, hi


def _gate_groups(rows, gates):
    """How many gates there are, gates = the shape of their tensor and rows = that of the input, both without the width; None if they are
    not each for a run of neighbouring rows."""
    count, all_rows = math.prod(gates), math.prod(rows)
    if len(rows) <= 1:                           # rows without a structure
        return count if all_rows == 0 or count and all_rows % count == 0 else None
    if count == 1 or (len(gates) == 1 and count == all_rows):
        return count
    while len(gates) > len(rows) and gates[0] == 1:
        gates = gates[1:]
    # leading axes of one may be left out
    ones = next((i for i, n in enumerate(rows) if n != 1), len(rows))
    for of in (rows, rows[ones:]):
        same = next((i for i, (g, r) in enumerate(zip(gates, of)) if g != r), min(len(gates), len(of)))
        if all(g == 1 for g in gates[same:]):
            return count
    return None


def _rows_in(inputs):
    if not torch.is_tensor(inputs) or inputs.dim() < 1:
        raise InvalidArgumentError("input must be a tensor of at least one dimension")


def _table_of(mul_map_file, num_bits):
    if int(num_bits) != 8:
        raise InvalidArgumentError("only num_bits = 8 is supported")
    return mul_map_file if isinstance(mul_map_file, TruthTable) else TruthTable(mul_map_file, num_bits)


class FakeApproxDense:
    """The layer call of FakeApproxConv2D around a matrix product: the ranges of the input and the kernel, fake quantization of
    both, the product with every 8x8-bit product looked up in the table, bias, activation; and a residual added behind that.

    inputs [..., depth] in float32, bfloat16 or float16; kernel [depth, columns] in any of them, or what pack() made of one;
    bias [columns] in any of them; residual and the output are like the input's type, [..., columns].

    activation: None, "relu", "gelu", "gelu_tanh" or "silu".  input_minmax: a range for all inputs, as from a calibration; by
    default every call finds its input's own, over all rows.  The kernel's range is always its own."""

    def __init__(self, mul_map_file, activation=None, num_bits=8, input_minmax=None):
        if activation not in _ACTIVATIONS:
            raise UnimplementedError("activation %r: only None, 'relu', 'gelu', 'gelu_tanh' and 'silu'" % (activation,))
        self.table = _table_of(mul_map_file, num_bits)
        self.activation = _ACTIVATIONS[activation]
        self.input_minmax = _minmax_of(input_minmax)
        self._descs = {}

    def _desc(self, inputs, depth, columns, kernel_dtype, bias):
        """[description, reference to it, output's shape, whether a call of a packed kernel is known to need no workspace] of a call:
        made once for its shapes and types."""
        key = (inputs.shape, inputs.dtype, depth, columns, kernel_dtype, None if bias is None else bias.dtype, self.activation,
               self.input_minmax)
        found = self._descs.get(key)
        if found is None:
            desc = _dense_desc(inputs, depth, columns, kernel_dtype, bias, self.activation, self.input_minmax)
            found = [desc, ctypes.byref(desc), inputs.shape[:-1] + (columns,), False]
            if len(self._descs) >= 256:
                self._descs.clear()
            self._descs[key] = found
        return found

    def pack(self, kernel):
        """The kernel as codes, for calls with the same kernel."""
        lib = _lib.load()
        kernel = _kernel_of(kernel, None)
        depth, columns = kernel.shape
        desc = _lib.DenseDesc(0, depth, columns, _lib.F32, _TYPES[kernel.dtype], _lib.F32, 0, 0, 0.0, 0.0)
        nbytes = ctypes.c_size_t()
        _check(lib.axc_dense_packed_bytes(ctypes.byref(desc), ctypes.byref(nbytes)))
        data = torch.empty(nbytes.value, dtype=torch.uint8, device=kernel.device)
        _launch(kernel.device, lib.axc_dense_pack, ctypes.byref(desc), kernel.data_ptr(), data.data_ptr(), _stream(kernel.device))
        return PackedKernel(data, depth, columns, kernel.dtype)

    def __call__(self, inputs, kernel, bias=None, residual=None, input_range=None):
        """input_range: what ResidualNorm.call_in_turn or FakeApproxConv2D.call_in_turn reported of `inputs`, which the call then
        need not read to find its range."""
        return self._run(inputs, kernel, bias, residual, input_range, False)[0]

    def call_and_keep(self, inputs, kernel, bias=None, residual=None, input_range=None):
        """(output, what the activation was given): the second is what gradients() needs where there is an activation."""
        return self._run(inputs, kernel, bias, residual, input_range, True)

    def _run(self, inputs, kernel, bias, residual, input_range, keep):
        lib = _lib.load()
        _rows_in(inputs)
        _unrecorded(inputs, kernel, bias, residual)
        found = _range_pointer(input_range, inputs)
        inputs = _require(inputs, "input")
        device = inputs.device
        packed = isinstance(kernel, PackedKernel)
        if packed:
            depth, columns, kernel_dtype = kernel.depth, kernel.columns, kernel.dtype
            if kernel.data.device != device:
                raise InvalidArgumentError("kernel is on another device than the input")
        else:
            kernel = _kernel_of(kernel, device)
            (depth, columns), kernel_dtype = kernel.shape, kernel.dtype
        if bias is not None:
            bias = _require(bias, "bias", device, shape=(columns,))
        call = self._desc(inputs, depth, columns, kernel_dtype, bias)
        _, ref, out_shape, bare = call
        if residual is not None:
            residual = _require(residual, "residual", device, inputs.dtype, out_shape)
        need, ws = 0, None
        if not (packed and bare):        # (what many rows need depends on the forms that are pinned; nothing, on the shape alone)
            nbytes = ctypes.c_size_t()
            _check(lib.axc_fake_approx_dense_workspace_bytes(ref, packed, ctypes.byref(nbytes)))
            need = nbytes.value
            ws = _scratch(need, device)
            call[3] = packed and need == 0
        out = torch.empty(out_shape, dtype=inputs.dtype, device=device)
        pre = torch.empty(out_shape, dtype=inputs.dtype, device=device) if keep else None
        _launch(device, lib.axc_fake_approx_dense, self.table.handle, ref, inputs.data_ptr(), found,
                None if packed else kernel.data_ptr(), kernel.data.data_ptr() if packed else None, _pointer(bias),
                _pointer(residual), out.data_ptr(), _pointer(pre), _pointer(ws), need, _stream(device))
        return out, pre

    def gradients(self, grad_output, inputs, kernel, pre=None, input_range=None, want=("inputs", "kernel", "bias")):
        """DenseGradients(inputs, kernel, bias) from the output's gradient, straight through the grid: a value inside its grid's
        range gets the gradient of the exact product of quantized values, one outside gets 0, and ranges count as constants.  The
        residual's gradient is grad_output itself; the bias' is of the kernel's type.  pre: what call_and_keep returned; without an
        activation it may be None.  want: which are made; the others are None."""
        lib = _lib.load()
        _rows_in(inputs)
        found = _range_pointer(input_range, inputs)
        inputs = _require(inputs, "input")
        device = inputs.device
        kernel = _kernel_of(kernel, device)
        depth, columns = kernel.shape
        if not set(want) <= {"inputs", "kernel", "bias"}:
            raise InvalidArgumentError("want: 'inputs', 'kernel', 'bias'")
        _, ref, out_shape, _ = self._desc(inputs, depth, columns, kernel.dtype, None)
        grad_output = _require(grad_output, "grad_output", device, inputs.dtype, out_shape)
        if pre is not None:
            pre = _require(pre, "pre", device, inputs.dtype, out_shape)
        nbytes = ctypes.c_size_t()
        _check(lib.axc_fake_approx_dense_gradients_workspace_bytes(ref, ctypes.byref(nbytes)))
        ws = _scratch(nbytes.value, device)
        dx = torch.empty_like(inputs) if "inputs" in want else None
        dk = torch.empty_like(kernel) if "kernel" in want else None
        db = torch.empty(columns, dtype=kernel.dtype, device=device) if "bias" in want else None
        _launch(device, lib.axc_fake_approx_dense_gradients, ref, grad_output.data_ptr(), inputs.data_ptr(), found,
                kernel.data_ptr(), _pointer(pre), _pointer(dx), _pointer(dk), _pointer(db), _pointer(ws), nbytes.value,
                _stream(device))
        return DenseGradients(dx, dk, db)


class FakeApproxCrossEntropy:
    """Softmax cross entropy of a FakeApproxDense layer's product + bias over a vocabulary (kernel [depth, vocabulary]), the logits
    made a piece of the vocabulary at a time and never kept.

    targets: int64 or int32, the input's shape without its last axis.  Rows whose target is ignore_index count for nothing but the
    input's range; a target that is no column of the vocabulary makes its row's loss NaN, and every gradient the row enters.
    reduction: "mean" (over the rows that count; 0 where none does), "sum" or "none"."""

    def __init__(self, mul_map_file, ignore_index=-100, num_bits=8, input_minmax=None):
        self.table = _table_of(mul_map_file, num_bits)
        self.ignore_index = int(ignore_index)
        self.input_minmax = _minmax_of(input_minmax)

    def __call__(self, inputs, kernel, targets, bias=None, reduction="mean", input_range=None):
        """The loss, in float32."""
        _unrecorded(inputs, kernel, bias)
        return self._run(inputs, kernel, targets, bias, reduction, None, input_range, ())[0]

    def loss_and_gradients(self, inputs, kernel, targets, bias=None, reduction="mean", grad_loss=None, input_range=None,
                           want=("inputs", "kernel", "bias")):
        """(loss, DenseGradients) of the loss times grad_loss (a float32 tensor like the loss; None: ones), straight through the grid
        as FakeApproxDense.gradients.  The bias' gradient is of the kernel's type, and None without a bias."""
        if not set(want) <= {"inputs", "kernel", "bias"}:
            raise InvalidArgumentError("want: 'inputs', 'kernel', 'bias'")
        return self._run(inputs, kernel, targets, bias, reduction, grad_loss, input_range, want)

    def _run(self, inputs, kernel, targets, bias, reduction, grad_loss, input_range, want):
        lib = _lib.load()
        _rows_in(inputs)
        found = _range_pointer(input_range, inputs)
        inputs = _require(inputs, "input")
        device = inputs.device
        kernel = _kernel_of(kernel, device)
        depth, columns = kernel.shape
        if bias is not None:
            bias = _require(bias, "bias", device, shape=(columns,))
        if reduction not in _REDUCTIONS:
            raise InvalidArgumentError("reduction must be 'none', 'sum' or 'mean'")
        if not torch.is_tensor(targets) or targets.device != device or targets.dtype not in (torch.int64, torch.int32):
            raise InvalidArgumentError("targets must be an int64 or int32 tensor on the input's GPU")
        if targets.shape != inputs.shape[:-1]:
            raise InvalidArgumentError("targets must have the shape %s" % (tuple(inputs.shape[:-1]),))
        targets = targets.to(torch.int64).contiguous()
        loss_shape = targets.shape if reduction == "none" else ()
        if grad_loss is not None:
            grad_loss = _require(grad_loss, "grad_loss", device, torch.float32, loss_shape)
        desc = _dense_desc(inputs, depth, columns, kernel.dtype, bias, 0, self.input_minmax)
        ref = ctypes.byref(desc)
        dx = torch.empty_like(inputs) if "inputs" in want else None
        dk = torch.empty_like(kernel) if "kernel" in want else None
        db = torch.empty(columns, dtype=kernel.dtype, device=device) if "bias" in want and bias is not None else None
        nbytes = ctypes.c_size_t()
        gradients = not (dx is None and dk is None and db is None)
        _check(lib.axc_fake_approx_cross_entropy_workspace_bytes(ref, gradients, ctypes.byref(nbytes)))
        ws = _scratch(nbytes.value, device)
        loss = torch.empty(loss_shape, dtype=torch.float32, device=device)
        _launch(device, lib.axc_fake_approx_cross_entropy, self.table.handle, ref, inputs.data_ptr(), found, kernel.data_ptr(),
                _pointer(bias), targets.data_ptr(), self.ignore_index, _REDUCTIONS[reduction], _pointer(grad_loss), loss.data_ptr(),
                _pointer(dx), _pointer(dk), _pointer(db), _pointer(ws), nbytes.value, _stream(device))
        return loss, DenseGradients(dx, dk, db)


class ResidualNorm:
    """The norms before and after a block of a residual network, with the block's gate and scale:

        u = norm(block) * post_weight, or block itself without post_weight
        h = x + scale * gate * u
        y = norm(h) * weight + bias

    norm: kind "rms" (v / sqrt(mean(v^2) + eps)) or "layer" ((v - mean) / sqrt(var + eps)).  x, block, gate and the outputs are of
    one type (float32, bfloat16, float16); weight, bias, scale, post_weight [width] of one type, any of them.  gate: [..., width],
    each for a run of neighbouring rows: one for all, one for every row, or the input's leading axes, with nothing but ones behind them
    ([batch, width] or [batch, 1, width] against [batch, tokens, width]); against an input [rows, width] any number that divides the
    rows.  Gates that would go round faster than the rows ([tokens, width] or [1, tokens, width]) are refused: expand them.  Without
    a block h is x."""

    def __init__(self, kind="rms", eps=1e-6):
        if kind not in _NORMS:
            raise UnimplementedError("norm %r: only 'rms' and 'layer'" % (kind,))
        if not 0.0 <= float(eps) < float("inf"):
            raise InvalidArgumentError("eps must be a number that is not negative")
        self.kind, self.eps = _NORMS[kind], float(eps)

    def _tensors(self, like, block, weight, bias, gate, scale, post_weight):
        """(desc, tensors for the call, what keeps them alive)"""
        device, width = like.device, like.shape[-1]
        rows = like.numel() // width if width else 0
        if block is not None:
            block = _require(block, "block", device, like.dtype, like.shape)
        elif gate is not None or scale is not None or post_weight is not None:
            raise InvalidArgumentError("gate, scale and post_weight need a block")
        weight = _require(weight, "weight", device, shape=(width,))
        vectors = [v if v is None else _require(v, what, device, weight.dtype, (width,))
                   for v, what in ((bias, "bias"), (scale, "scale"), (post_weight, "post_weight"))]
        groups = 0
        if gate is not None:
            gate = _require(gate, "gate", device, like.dtype)
            if gate.dim() < 1 or gate.shape[-1] != width:
                raise InvalidArgumentError("gate must be as wide as the input")
            groups = _gate_groups(tuple(like.shape[:-1]), tuple(gate.shape[:-1]))
            if groups is None:
                raise InvalidArgumentError("a gate %s is not one for each of a number of runs of rows of an input %s" %
                                           (tuple(gate.shape), tuple(like.shape)))
        desc = _lib.ResidualNormDesc(rows, width, groups, _TYPES[like.dtype], _TYPES[weight.dtype], self.kind, self.eps)
        alive = [None, block, weight, vectors[0], gate, vectors[1], vectors[2]]
        return desc, alive

    def __call__(self, x, block, weight, bias=None, gate=None, scale=None, post_weight=None):
        """(h, y)"""
        return self._run(x, block, weight, bias, gate, scale, post_weight, False)[:2]

    def call_in_turn(self, x, block, weight, bias=None, gate=None, scale=None, post_weight=None):
        """(h, y, range): the third for the input_range of a FakeApproxDense or FakeApproxConv2D call on that very y, which then
        need not read it to find its smallest and largest value."""
        h, y, seen = self._run(x, block, weight, bias, gate, scale, post_weight, True)
        if seen is not None:
            seen._range_of = weakref.ref(y), _version(y)
        return h, y, seen

    def _run(self, x, block, weight, bias, gate, scale, post_weight, want_range):
        lib = _lib.load()
        _rows_in(x)
        _unrecorded(x, block, weight, bias, gate, scale, post_weight)
        x = _require(x, "x")
        desc, alive = self._tensors(x, block, weight, bias, gate, scale, post_weight)
        alive[0] = x
        device = x.device
        y = torch.empty_like(x)
        h = torch.empty_like(x) if block is not None else x
        seen = None
        if want_range and desc.rows:
            seen = torch.empty(_lib.RANGE_BYTES // 4, dtype=torch.float32, device=device)
        tensors = _lib.ResidualNormTensors(*[_pointer(t) for t in alive])
        _launch(device, lib.axc_residual_norm, ctypes.byref(desc), ctypes.byref(tensors), h.data_ptr(), y.data_ptr(), _pointer(seen),
                _stream(device))
        return h, y, seen

    def gradients(self, grad_h, grad_y, h, block, weight, bias=None, gate=None, scale=None, post_weight=None):
        """ResidualNormGradients from those of h and y (one of them may be None: zeros) and what the call was given, h as it
        returned it.  Gradients of what is None are None."""
        lib = _lib.load()
        _rows_in(h)
        h = _require(h, "h")
        desc, alive = self._tensors(h, block, weight, bias, gate, scale, post_weight)
        device = h.device
        if grad_h is None and grad_y is None:
            raise InvalidArgumentError("the gradient of h or of y")
        grad_h, grad_y = (g if g is None else _require(g, what, device, h.dtype, h.shape)
                          for g, what in ((grad_h, "grad_h"), (grad_y, "grad_y")))
        out = [torch.empty_like(h)] + [None if t is None else torch.empty_like(t) for t in alive[1:]]
        nbytes = ctypes.c_size_t()
        ref = ctypes.byref(desc)
        _check(lib.axc_residual_norm_gradients_workspace_bytes(ref, ctypes.byref(nbytes)))
        ws = _scratch(nbytes.value, device)
        tensors = _lib.ResidualNormTensors(*[_pointer(t) for t in alive])
        outs = _lib.ResidualNormTensors(*[_pointer(t) for t in out])
        _launch(device, lib.axc_residual_norm_gradients, ref, ctypes.byref(tensors), h.data_ptr(), _pointer(grad_h), _pointer(grad_y),
                ctypes.byref(outs), _pointer(ws), nbytes.value, _stream(device))
        return ResidualNormGradients(*out)
