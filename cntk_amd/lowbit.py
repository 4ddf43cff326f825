"""Low-bit training and serving of linear layers on one MI355X: products of matrices in 4-bit microscaled form, activations kept for
the backward pass in 8 bits, and the weight gradient read from what was kept -- which the gradient quantizer of this package
(`torch_hook.QuantizedGradientAggregator`) then aggregates.

    q = mx4_quantize(w)                      a matrix in 4-bit form, blocks of 32 along its rows; mx4_quantize(w.t()) for the other way
    y = mx4_linear(x, q, bias)               x W' + b, x put into 4 bits on the way; any number of rows, few of them in one launch
    y, kept = mx4_linear(x, q, bias, save=True)      ... and x kept in 8 bits from the same reading of it
    y, kept = activation_forward("silu", x, gate)    f(x), or f(gate) x, with its inputs kept in 8 bits
    dx = activation_backward(dy, kept)       (dx, dgate) for a gated one
    dw, db = weight_gradient(dy, kept, bias=True)    dy' x and the column sums of dy, in 32 bits

`LowBitLinear` and `LowBitActivation` are these as torch modules. The formats, and what becomes of infinities and NaN, are described in
``include/cntk_amd_lowbit.h``.

Element types: float32, float16, bfloat16. Tensors of more than two dimensions are taken as rows of their last one. Everything is issued
on torch's current stream of the tensors' device; nothing waits and nothing is kept between calls. As with any torch operator, a tensor made on
another stream needs that stream's work to be over or waited for. The functions take part in no autograd graph; the modules do. An `out` that
requires grad is refused while gradients are recorded, and so is one that shares memory with another tensor of the call; what is written raises its version, so that a backward pass that needs the old values says so.
Errors are this package's: QuantizerLogicError for arguments that do not fit, QuantizerError for a failed device call.
"""
import ctypes
import importlib.util
import os

import torch

from . import QuantizerError, QuantizerLogicError, lib as _base_lib

_sz, _vp, _i64, _int = ctypes.c_size_t, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTIVATIONS = {"sigmoid": 1, "tanh": 2, "relu": 3, "gelu": 4, "silu": 5}

_lib = None


def _bind():
    """The library with the low-bit calls' argument types, for callers of the C ABI."""
    global _lib
    L = _base_lib()
    for name in ("cntkq_mx4_bytes", "cntkq_save8_bytes"):
        getattr(L, name).argtypes, getattr(L, name).restype = [_sz, _sz], _sz
    L.cntkq_mx4_linear_workspace_bytes.argtypes, L.cntkq_mx4_linear_workspace_bytes.restype = [_sz, _sz, _sz, _int, _int], _sz
    L.cntkq_weight_gradient_workspace_bytes.argtypes, L.cntkq_weight_gradient_workspace_bytes.restype = [_sz, _sz, _sz, _int], _sz
    L.cntkq_mx4_quantize_async.argtypes = [_vp, _vp, _int, _sz, _sz, _i64, _i64, _vp, _sz, _vp, _sz]
    L.cntkq_mx4_dequantize_async.argtypes = [_vp, _vp, _sz, _sz, _sz, _vp, _int, _i64]
    L.cntkq_mx4_matmul_async.argtypes = [_vp, _vp, _sz, _sz, _vp, _sz, _sz, _sz, _vp, _int, _vp, _int, _i64]
    L.cntkq_mx4_linear_async.argtypes = [_vp, _vp, _int, _i64, _sz, _vp, _sz, _sz, _sz, _vp, _int, _vp, _int, _i64, _vp, _sz, _vp, _sz]
    L.cntkq_save8_async.argtypes = [_vp, _vp, _int, _sz, _sz, _i64, _vp, _sz]
    L.cntkq_load8_async.argtypes = [_vp, _vp, _sz, _sz, _sz, _vp, _int, _i64]
    L.cntkq_activation_forward_async.argtypes = [_vp, _int, _vp, _i64, _vp, _i64, _int, _sz, _sz, _vp, _i64, _vp, _vp, _sz]
    L.cntkq_activation_backward_async.argtypes = [_vp, _int, _vp, _i64, _int, _sz, _sz, _vp, _vp, _sz, _vp, _i64, _vp, _i64]
    L.cntkq_weight_gradient_async.argtypes = [_vp, _vp, _int, _i64, _sz, _sz, _vp, _sz, _sz, _vp, _i64, _vp, _int, _vp, _sz]
    _lib = L
    return L


def _load_binding():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lowbit.so")
    if not os.path.exists(path):
        raise ImportError("%s is missing: build it with `python -m cntk_amd.build` (there is no fallback)" % path)
    spec = importlib.util.spec_from_file_location("cntk_amd._lowbit", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.errors(QuantizerError, QuantizerLogicError)
    return module


_ops = _load_binding()  # csrc/lowbit_torch.cpp: checks the tensors, makes the results, calls the C ABI


def _type(dtype):
    code = _DTYPES.get(dtype)
    if code is None:
        raise QuantizerLogicError("dtype must be float32, float16 or bfloat16")
    return code


class Mx4Matrix:
    """A matrix in 4-bit microscaled form, packed in `buffer` (uint8, on the device)."""
    __slots__ = ("rows", "cols", "buffer")

    def __init__(self, rows, cols, buffer=None, device="cuda:0"):
        rows, cols = int(rows), int(cols)
        size = (_lib or _bind()).cntkq_mx4_bytes(rows, cols)
        if buffer is None:
            buffer = torch.empty(size, dtype=torch.uint8, device=device)
        elif buffer.dtype != torch.uint8 or buffer.dim() != 1 or buffer.numel() != size or not buffer.is_cuda or not buffer.is_contiguous():
            raise QuantizerLogicError("the buffer of a %d x %d matrix in 4 bits is a flat uint8 device tensor of %d elements" % (rows, cols, size))
        self.rows, self.cols, self.buffer = rows, cols, buffer

    @classmethod
    def _of(cls, buffer, rows, cols):
        q = cls.__new__(cls)
        q.buffer, q.rows, q.cols = buffer, rows, cols
        return q

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self):
        return self.buffer.device


class Saved8:
    """What was kept in 8 bits: an input of `shape` (`buffer`), a gate of the same shape or None (`gate`), and the
    activation's name they go through or None."""
    __slots__ = ("shape", "dtype", "buffer", "gate", "kind")

    def __init__(self, shape, dtype, buffer, gate=None, kind=None):
        self.shape, self.dtype, self.buffer, self.gate, self.kind = torch.Size(shape), dtype, buffer, gate, kind

    @property
    def cols(self):
        return self.shape[-1]

    @property
    def rows(self):
        return self.shape[:-1].numel()

    def values(self, dtype=None):
        """The kept input's values (a pair with the gate's where there is one), in `dtype` or the input's own type."""
        code = _type(dtype or self.dtype)
        made = [_ops.load8(b, self.rows, self.cols, code).view(self.shape) for b in (self.buffer, self.gate) if b is not None]
        return made[0] if len(made) == 1 else tuple(made)


# ---- 4 bits ---------------------------------------------------------------------------------------


def mx4_quantize(x, out=None):
    """x in 4-bit form, blocks along its last dimension. A matrix may have any strides: mx4_quantize(x.t()) has the blocks along the
    other axis. out: an Mx4Matrix of x's shape to write into."""
    if out is not None:
        rows = x.numel() // max(x.shape[-1], 1) if x.dim() else 0
        if not x.dim() or x.shape[-1] != out.cols or rows != out.rows:
            raise QuantizerLogicError("out is a %d x %d matrix, x of shape %s" % (out.rows, out.cols, tuple(x.shape)))
        _ops.quantize(x, out.buffer)
        return out
    return Mx4Matrix._of(*_ops.quantize(x, None))


def mx4_dequantize(q, dtype=torch.bfloat16, out=None):
    """The values of a matrix in 4-bit form (bfloat16 and float32 hold all of them)."""
    return _ops.dequantize(q.buffer, q.rows, q.cols, _type(dtype), out)


def mx4_matmul(a, b, bias=None, dtype=torch.bfloat16, out=None):
    """a b' (+ bias) of two matrices in 4-bit form: a m x k, b n x k, the result m x n. Sums in 32 bits, rounded once."""
    if a.cols != b.cols:
        raise QuantizerLogicError("the inner sides differ: %d and %d" % (a.cols, b.cols))
    return _ops.matmul(a.buffer, a.rows, b.buffer, b.rows, a.cols, bias, _type(dtype), out)


def mx4_linear(x, weight, bias=None, save=False, dtype=None, out=None):
    """x W' (+ bias) with x put into 4-bit form on the way: what mx4_matmul(mx4_quantize(x), weight, bias) gives, up to the order of
    the sums. The result has x's type unless `dtype` names another. save: also returns x kept in 8 bits (Saved8), for weight_gradient."""
    made = _ops.linear(x, weight.buffer, weight.rows, weight.cols, bias, save, -1 if dtype is None else _type(dtype), out)
    return (made[0], Saved8(x.shape, x.dtype, made[1])) if save else made


# ---- 8 bits ---------------------------------------------------------------------------------------


def save8(x):
    """x kept in 8 bits (Saved8)."""
    return Saved8(x.shape, x.dtype, _ops.save8(x))


def activation_forward(kind, x, gate=None):
    """(f(x), kept), or (f(gate) x, kept) with a gate of x's shape; kind: one of ACTIVATIONS. The function is taken of the inputs as they
    are; `kept` (Saved8) holds them in 8 bits for activation_backward."""
    number = ACTIVATIONS.get(kind)
    if number is None:
        raise QuantizerLogicError("unknown activation %r: one of %s" % (kind, ", ".join(ACTIVATIONS)))
    y, saved, saved_gate = _ops.activation_forward(number, x, gate)
    return y, Saved8(x.shape, x.dtype, saved, saved_gate, kind)


def activation_backward(dy, kept):
    """The gradient of the activation's input, dy f'(x8), from what activation_forward kept; (dx, dgate) for a gated one:
    dy f(g8) and dy x8 f'(g8)."""
    if kept.kind is None:
        raise QuantizerLogicError("what was kept has not gone through an activation")
    if dy.shape != kept.shape or dy.dtype != kept.dtype:
        raise QuantizerLogicError("dy must be of the kept input's shape and type, on its device")
    return _ops.activation_backward(ACTIVATIONS[kept.kind], dy, kept.buffer, kept.gate)


def weight_gradient(dy, kept, bias=False, out=None, accumulate=False):
    """dw = dy' x8 (n x k, float32) from the layer's input as kept (save8, mx4_linear(save=True)); with bias=True (dw, db), db the column
    sums of dy. out: dw, or the pair (dw, db), to write into, either of them None for a new tensor; accumulate: added to what they hold, both
    given then."""
    if kept.kind is not None:
        raise QuantizerLogicError("what was kept belongs to an activation")
    if dy.shape[:-1] != kept.shape[:-1]:
        raise QuantizerLogicError("dy has other rows (%s) than the kept input (%s)" % (tuple(dy.shape), tuple(kept.shape)))
    dw, db = (None, None) if out is None else (out if bias else (out, None))
    return _ops.weight_gradient(dy, kept.buffer, kept.shape[-1], bias, dw, db, accumulate)


# ---- torch modules --------------------------------------------------------------------------------


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        q = mx4_quantize(weight)
        keep = weight.requires_grad or (bias is not None and bias.requires_grad)
        made = mx4_linear(x, q, bias, save=keep)
        y, kept = made if keep else (made, None)
        q_t = mx4_quantize(weight.t()) if x.requires_grad else None
        ctx.save_for_backward(None if kept is None else kept.buffer, None if q_t is None else q_t.buffer)
        ctx.x_shape, ctx.x_dtype, ctx.out_features = x.shape, x.dtype, weight.shape[0]
        ctx.types = weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        kept, q_t = ctx.saved_tensors
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = mx4_linear(dy, Mx4Matrix._of(q_t, ctx.x_shape[-1], ctx.out_features))
        if kept is not None:
            with_bias = ctx.types[1] is not None
            dw = weight_gradient(dy, Saved8(ctx.x_shape, ctx.x_dtype, kept), bias=with_bias)
            if with_bias:
                dw, db = dw
                db = db.to(ctx.types[1])
            dw = dw.to(ctx.types[0])
        return dx, dw, db


class _ActivationFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, kind, x, gate):
        y, kept = activation_forward(kind, x, gate)
        ctx.save_for_backward(kept.buffer, kept.gate)
        ctx.x_shape, ctx.x_dtype, ctx.kind = x.shape, x.dtype, kind
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        buffer, gate = ctx.saved_tensors
        d = activation_backward(dy, Saved8(ctx.x_shape, ctx.x_dtype, buffer, gate, ctx.kind))
        return (None,) + (d if gate is not None else (d, None))


class LowBitLinear(torch.nn.Module):
    """torch.nn.Linear with its product in 4 bits and its input kept in 8. The weights are an ordinary parameter (float32 unless asked
    otherwise) and are put into 4-bit form, in both directions, at every forward pass; `freeze` does that once, for serving."""

    def __init__(self, in_features, out_features, bias=True, device=None, dtype=None):
        super().__init__()
        like = torch.nn.Linear(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.in_features, self.out_features = in_features, out_features
        self.weight, self.bias = like.weight, like.bias
        self._frozen = None

    def freeze(self):
        """Keeps the weights as they are now in 4 bits; forward passes use them, without gradients, until unfreeze()."""
        self._frozen = mx4_quantize(self.weight.detach())
        return self

    def unfreeze(self):
        self._frozen = None
        return self

    def forward(self, x):
        if self._frozen is not None:
            return mx4_linear(x.detach(), self._frozen, None if self.bias is None else self.bias.detach())
        return _LinearFunction.apply(x, self.weight, self.bias)


class LowBitActivation(torch.nn.Module):
    """f(x), or f(gate) x, with its inputs kept in 8 bits for the backward pass."""

    def __init__(self, kind):
        super().__init__()
        if kind not in ACTIVATIONS:
            raise QuantizerLogicError("unknown activation %r: one of %s" % (kind, ", ".join(ACTIVATIONS)))
        self.kind = kind

    def forward(self, x, gate=None):
        return _ActivationFunction.apply(self.kind, x, gate)
