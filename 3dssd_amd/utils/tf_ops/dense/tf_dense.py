"""The dense layer (a 1x1 convolution, a fully connected layer) on plain weights, and its gradient, on torch-ROCm tensors,
backed by the gfx950 kernels behind include/sa_ops.h (csrc/dense.hip).

The layers of the detector itself run `sa_dense` on BN-folded, packed inference weights (utils/weights.py).  These two
functions are for weights as a training step or a serving loop holds them: `[cin, cout]` in fp32, bf16 or fp16, with bias,
activation and residual in the product's epilogue, and with a backward pass.  Like the other gradients of this package
(`group_point_grad`, `gather_point_grad`) it is an explicit function: nothing is registered with autograd.

    z = inputs @ weights + biases,   out = activation(z) + residual

fp32 in, fp32 arithmetic; bf16 / fp16 in, fp32 sums, each output rounded once.  Large fp32 layers take their factors apart into
bf16 planes: a factor is held to 2^-24 of itself or to 2^-134, whichever is larger (below 2^-110 that is fewer than 24 bits:
scale such operands by a power of two), and a sum within a hundredth of the largest fp32 number may become infinite.
"""
import ctypes
import functools
import math

import torch

from .. import _tensor as T
from ... import _native as N

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_ROUND_SLOPES = 16                    # added to the activation's number
_FAR = 1 << 24                        # rows further apart than this are copied together; longer ones are refused


def _operand(t, name, dtype=None):
    """Raises unless t is a tensor the kernels can read."""
    T.require(isinstance(t, torch.Tensor), "%s must be a torch.Tensor" % name)
    T.require(t.is_cuda, "%s must live on the GPU (the HIP path has no CPU fallback)" % name)
    T._on_current_device(t, name)
    T.require(t.dtype in TYPES, "%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))
    T.require(dtype is None or t.dtype == dtype, "%s is %s but inputs are %s" % (name, t.dtype, dtype))


def _beside(t, name, inputs, *dtypes):
    """Raises unless t is a tensor beside inputs, of its type (or one of dtypes)."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == inputs.get_device() and
            (t.dtype == inputs.dtype or t.dtype in dtypes)):
        _operand(t, name, None if dtypes else inputs.dtype)
        raise ValueError("%s must be float32 or of the inputs' type" % name)


def _rows(t, cols):
    """[..., cols] as (tensor, address, elements between rows) with the columns contiguous; a view where the strides allow
    it, a copy otherwise."""
    m = t if t.dim() == 2 else t.reshape(-1, cols) if cols else t.reshape(math.prod(t.shape[:-1]), 0)
    rows = m.shape[0]
    ld, step = m.stride()
    if (step != 1 and cols > 1) or ((ld < cols or ld >= _FAR) and rows > 1):
        m = m.contiguous()
        ld = cols
    return m, m.data_ptr(), (ld if rows > 1 else cols)


@functools.lru_cache(maxsize=4096)
def _forward_ws(*args):
    n = ctypes.c_ulong()
    N.check(N.lib().sa_dense_forward_ws(*args, ctypes.byref(n)), "dense")
    return n.value


@functools.lru_cache(maxsize=4096)
def _backward_ws(*args):
    n = ctypes.c_ulong()
    N.check(N.lib().sa_dense_backward_ws(*args, ctypes.byref(n)), "dense_grad")
    return n.value


def _layer(op, inputs, weights, biases, activation):
    """Checks what both functions take; (type, cin, cout, device).  One pass over the conditions in the ordinary case: the
    messages are only made where one of them does not hold."""
    if not (isinstance(inputs, torch.Tensor) and isinstance(weights, torch.Tensor) and inputs.is_cuda and
            inputs.get_device() == weights.get_device() == torch._C._cuda_getDevice() and
            inputs.dtype == weights.dtype and inputs.dtype in TYPES):
        _operand(inputs, "inputs")
        _operand(weights, "weights", inputs.dtype)
    if activation not in ACTIVATIONS:
        raise ValueError("%s knows the activations %s, not %r" % (op, sorted(a for a in ACTIVATIONS if a), activation))
    if weights.dim() != 2:
        raise ValueError("%s expects (cin,cout) weights shape" % op)
    cin, cout = weights.shape
    if inputs.dim() == 0 or inputs.size(-1) != cin:
        raise ValueError("%s expects (...,cin) inputs shape" % op)
    if cin >= _FAR or cout >= _FAR:
        raise ValueError("%s expects fewer than 2**24 channels" % op)
    if biases is not None:
        _beside(biases, "biases", inputs, torch.float32)
        if biases.dim() != 1 or biases.size(0) != cout:
            raise ValueError("%s expects (cout) biases shape" % op)
    return inputs.dtype, cin, cout


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device)


def _aligned(ptr, ld, itemsize):
    return ptr % 16 == 0 and ld * itemsize % 16 == 0 and ld * itemsize < 1 << 22


def dense(inputs, weights, biases=None, activation=None, residual=None, return_preact=False):
    """activation(inputs @ weights + biases) + residual.

    inputs [..., cin], weights [cin, cout], biases [cout] or None, residual [..., cout] or None, all float32, bfloat16 or
    float16 and all of one type (biases may be float32 beside 16-bit inputs).  activation: None, "relu", "gelu" (with the
    normal integral), "gelu_tanh" or "silu".  Returns out [..., cout]; with return_preact also z [..., cout], which
    dense_grad needs.  Rows may lie apart (any stride, last dimension contiguous); other layouts are copied first.
    An input of no rows gives an empty result; with cin = 0 the product is zero."""
    dt, cin, cout = _layer("Dense", inputs, weights, biases, activation)
    shape = (inputs.size(0), cout) if inputs.dim() == 2 else inputs.shape[:-1] + (cout,)
    if residual is not None:
        _beside(residual, "residual", inputs)
        T.require(residual.shape == shape, "Dense expects (...,cout) residual shape")
    out = inputs.new_empty(shape)
    pre = inputs.new_empty(shape) if return_preact else None
    rows = out.numel() // cout if cout else 0
    if rows:
        x, xp, ldx = _rows(inputs, cin)
        w, wp, ldw = _rows(weights, cout)
        r, rp, ldr = (None, None, 0) if residual is None else _rows(residual, cout)
        b = None if biases is None else biases.contiguous()
        code, e = TYPES[dt], dt.itemsize
        need = _forward_ws(code, rows, cin, cout, _aligned(xp, ldx, e) + 2 * _aligned(wp, ldw, e))
        ws = inputs.new_empty(need, dtype=torch.uint8) if need else None
        N.check(N.lib().sa_dense_forward(code, rows, cin, cout, xp, ldx, wp, ldw, None if b is None else b.data_ptr(),
                                         int(b is not None and b.dtype == torch.float32), rp, ldr, ACTIVATIONS[activation],
                                         out.data_ptr(), None if pre is None else pre.data_ptr(),
                                         None if ws is None else ws.data_ptr(), need, _stream(inputs.get_device())), "dense")
    return (out, pre) if return_preact else out


def dense_grad(inputs, weights, grad_out, biases=None, activation=None, preact=None, needs=(True, True), round_slopes=False):
    """Gradient of dense: (grad_inputs [..., cin], grad_weights [cin, cout], grad_biases [cout]).

    grad_out [..., cout] is the gradient of dense's out (and, unchanged, the gradient of its residual); preact is the z that
    dense(..., return_preact=True) returned, needed with an activation.  ReLU's slope at 0 is 0.  needs: whether the first
    two are wanted (None in their place if not); grad_biases is computed where biases are given and has their type.
    With GELU or SiLU the 16-bit forms take grad_out * slope into both products in two planes of the type (to 2^-16 of itself in
    bf16, 2^-22 or 2^-35 in fp16), which is twice the products of the forward pass each.  round_slopes=True rounds it once to
    the type instead: up to half the time, and results with 1.4 times the relative error (2-norm) that rounding them alone
    makes.  The bias gradient sums it unrounded either way.
    Sums run in fp32 in a fixed order: the same call gives the same bits."""
    dt, cin, cout = _layer("DenseGrad", inputs, weights, biases, activation)
    shape = inputs.shape[:-1] + (cout,)
    _beside(grad_out, "grad_out", inputs)
    T.require(grad_out.shape == shape, "DenseGrad expects (...,cout) grad_out shape")
    if activation is None:
        preact = None
    else:
        T.require(preact is not None, "DenseGrad needs preact where there is an activation")
        _beside(preact, "preact", inputs)
        T.require(preact.shape == shape, "DenseGrad expects (...,cout) preact shape")
    T.require(len(needs) == 2, "needs: (inputs, weights)")
    dx = inputs.new_empty(inputs.shape) if needs[0] else None
    dw = inputs.new_empty((cin, cout)) if needs[1] else None
    db = biases.new_empty((cout,)) if biases is not None else None
    rows = 1
    for d in inputs.shape[:-1]:
        rows *= d
    x, xp, ldx = _rows(inputs, cin) if rows and cin else (None, None, cin)
    w, wp, ldw = _rows(weights, cout) if cin and cout else (None, None, cout)
    g, gp, ldg = _rows(grad_out, cout) if rows and cout else (None, None, cout)
    z, zp, ldz = _rows(preact, cout) if preact is not None and rows and cout else (None, None, cout)
    code, e, act = TYPES[dt], dt.itemsize, ACTIVATIONS[activation] + (_ROUND_SLOPES if round_slopes else 0)
    want = ((1 if dx is not None and rows and cin else 0) | (2 if dw is not None and cin and cout else 0)
            | (4 if db is not None and cout else 0))
    if want:
        aligned = sum(1 << i for i, (p, ld) in enumerate(((xp, ldx), (wp, ldw), (gp, ldg))) if p and _aligned(p, ld, e))
        need = _backward_ws(code, rows, cin, cout, act, want, aligned)
        ws = inputs.new_empty(need, dtype=torch.uint8) if need else None
        N.check(N.lib().sa_dense_backward(code, rows, cin, cout, xp, ldx, wp, ldw, gp, ldg, zp, ldz, act,
                                          dx.data_ptr() if want & 1 else None, dw.data_ptr() if want & 2 else None,
                                          db.data_ptr() if want & 4 else None, int(db is not None and db.dtype == torch.float32),
                                          None if ws is None else ws.data_ptr(), need, _stream(inputs.get_device())), "dense_grad")
    return dx, dw, db
