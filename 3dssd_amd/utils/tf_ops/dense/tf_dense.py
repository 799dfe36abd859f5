"""The dense layer (a 1x1 convolution, a fully connected layer) on plain weights, and its gradient, on torch-ROCm tensors,
backed by the gfx950 kernels behind include/sa_ops.h (csrc/dense.hip).

The layers of the detector itself run `sa_dense` on BN-folded, packed inference weights (utils/weights.py).  These two
functions are for weights as a training step or a serving loop holds them: `[cin, cout]` in fp32, bf16 or fp16, with bias,
activation and residual in the product's epilogue, and with a backward pass.  Like the other gradients of this package
(`group_point_grad`, `gather_point_grad`) it is an explicit function: nothing is registered with autograd.

    z = inputs @ weights + biases,   out = activation(z) + residual

fp32 in, fp32 arithmetic; bf16 / fp16 in, fp32 sums, each output rounded once.
"""
import ctypes
import functools

import torch

from .. import _tensor as T
from ... import _native as N

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_MAX_CHANNELS = (1 << 31) - 1


def _operand(t, name, dtype=None):
    T.require(isinstance(t, torch.Tensor), "%s must be a torch.Tensor" % name)
    T.require(t.is_cuda, "%s must live on the GPU (the HIP path has no CPU fallback)" % name)
    T._on_current_device(t, name)
    T.require(t.dtype in TYPES, "%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))
    T.require(dtype is None or t.dtype == dtype, "%s is %s but inputs are %s" % (name, t.dtype, dtype))
    return t


def _rows(t, cols):
    """[..., cols] as (tensor, address, elements between rows) with the columns contiguous; a view where the strides allow
    it, a copy otherwise."""
    m = t if t.dim() == 2 else t.reshape(-1, cols)
    rows = m.shape[0]
    if cols > 1 and m.stride(1) != 1 or rows > 1 and m.stride(0) < cols:
        m = m.contiguous()
    return m, m.data_ptr(), (m.stride(0) if rows > 1 else cols)


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
    _operand(inputs, "inputs")
    dt = inputs.dtype
    _operand(weights, "weights", dt)
    T.require(activation in ACTIVATIONS, "%s knows the activations %s, not %r" % (op, sorted(a for a in ACTIVATIONS if a), activation))
    T.require(weights.dim() == 2, "%s expects (cin,cout) weights shape" % op)
    T.require(inputs.dim() >= 1 and inputs.shape[-1] == weights.shape[0], "%s expects (...,cin) inputs shape" % op)
    cin, cout = weights.shape
    T.require(max(cin, cout) <= _MAX_CHANNELS, "%s expects fewer than 2**31 channels" % op)
    if biases is not None:
        _operand(biases, "biases")
        T.require(biases.dtype in (dt, torch.float32), "biases must be float32 or of the inputs' type")
        T.require(tuple(biases.shape) == (cout,), "%s expects (cout) biases shape" % op)
    return dt, cin, cout


def _aligned(ptr, ld, itemsize):
    return ptr % 16 == 0 and ld * itemsize % 16 == 0 and ld < 1 << 21


def dense(inputs, weights, biases=None, activation=None, residual=None, return_preact=False):
    """activation(inputs @ weights + biases) + residual.

    inputs [..., cin], weights [cin, cout], biases [cout] or None, residual [..., cout] or None, all float32, bfloat16 or
    float16 and all of one type (biases may be float32 beside 16-bit inputs).  activation: None, "relu", "gelu" (with the
    normal integral), "gelu_tanh" or "silu".  Returns out [..., cout]; with return_preact also z [..., cout], which
    dense_grad needs.  Rows may lie apart (any stride, last dimension contiguous); other layouts are copied first.
    An input of no rows gives an empty result; with cin = 0 the product is zero."""
    dt, cin, cout = _layer("Dense", inputs, weights, biases, activation)
    shape = inputs.shape[:-1] + (cout,)
    if residual is not None:
        _operand(residual, "residual", dt)
        T.require(residual.shape == shape, "Dense expects (...,cout) residual shape")
    out = torch.empty(shape, dtype=dt, device=inputs.device)
    pre = torch.empty_like(out) if return_preact else None
    rows = out.numel() // cout if cout else 0
    if rows:
        x, xp, ldx = _rows(inputs, cin)
        w, wp, ldw = _rows(weights, cout)
        r, rp, ldr = (None, None, 0) if residual is None else _rows(residual, cout)
        b = None if biases is None else biases.contiguous()
        code, e = TYPES[dt], dt.itemsize
        need = _forward_ws(code, rows, cin, cout, _aligned(xp, ldx, e) + 2 * _aligned(wp, ldw, e))
        ws = torch.empty(need, dtype=torch.uint8, device=inputs.device) if need else None
        N.check(N.lib().sa_dense_forward(code, rows, cin, cout, xp, ldx, wp, ldw, None if b is None else b.data_ptr(),
                                         int(b is not None and b.dtype == torch.float32), rp, ldr, ACTIVATIONS[activation],
                                         out.data_ptr(), None if pre is None else pre.data_ptr(),
                                         None if ws is None else ws.data_ptr(), need, N.current_stream()), "dense")
    return (out, pre) if return_preact else out


def dense_grad(inputs, weights, grad_out, biases=None, activation=None, preact=None, needs=(True, True)):
    """Gradient of dense: (grad_inputs [..., cin], grad_weights [cin, cout], grad_biases [cout]).

    grad_out [..., cout] is the gradient of dense's out (and, unchanged, the gradient of its residual); preact is the z that
    dense(..., return_preact=True) returned, needed with an activation.  ReLU's slope at 0 is 0.  needs: whether the first
    two are wanted (None in their place if not); grad_biases is computed where biases are given and has their type.
    With an activation the 16-bit forms round grad_out * slope once to the inputs' type, as an operand of both products; the
    bias gradient sums it unrounded.  Sums run in fp32 in a fixed order: the same call gives the same bits."""
    dt, cin, cout = _layer("DenseGrad", inputs, weights, biases, activation)
    shape = inputs.shape[:-1] + (cout,)
    _operand(grad_out, "grad_out", dt)
    T.require(grad_out.shape == shape, "DenseGrad expects (...,cout) grad_out shape")
    if activation is None:
        preact = None
    else:
        T.require(preact is not None, "DenseGrad needs preact where there is an activation")
        _operand(preact, "preact", dt)
        T.require(preact.shape == shape, "DenseGrad expects (...,cout) preact shape")
    T.require(len(needs) == 2, "needs: (inputs, weights)")
    dev = inputs.device
    dx = torch.empty(inputs.shape, dtype=dt, device=dev) if needs[0] else None
    dw = torch.empty((cin, cout), dtype=dt, device=dev) if needs[1] else None
    db = torch.empty((cout,), dtype=biases.dtype, device=dev) if biases is not None else None
    rows = 1
    for d in inputs.shape[:-1]:
        rows *= d
    x, xp, ldx = _rows(inputs, cin) if rows and cin else (None, None, cin)
    w, wp, ldw = _rows(weights, cout) if cin and cout else (None, None, cout)
    g, gp, ldg = _rows(grad_out, cout) if rows and cout else (None, None, cout)
    z, zp, ldz = _rows(preact, cout) if preact is not None and rows and cout else (None, None, cout)
    code, e, act = TYPES[dt], dt.itemsize, ACTIVATIONS[activation]
    want = ((1 if dx is not None and rows and cin else 0) | (2 if dw is not None and cin and cout else 0)
            | (4 if db is not None and cout else 0))
    if want:
        aligned = sum(1 << i for i, (p, ld) in enumerate(((xp, ldx), (wp, ldw), (gp, ldg))) if p and _aligned(p, ld, e))
        need = _backward_ws(code, rows, cin, cout, act, want, aligned)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        N.check(N.lib().sa_dense_backward(code, rows, cin, cout, xp, ldx, wp, ldw, gp, ldg, zp, ldz, act,
                                          dx.data_ptr() if want & 1 else None, dw.data_ptr() if want & 2 else None,
                                          db.data_ptr() if want & 4 else None, int(db is not None and db.dtype == torch.float32),
                                          None if ws is None else ws.data_ptr(), need, N.current_stream()), "dense_grad")
    return dx, dw, db
