"""The global norm of a list of gradients and clipping by it, on torch-ROCm tensors, backed by csrc/gradnorm.hip through the
C ABI of include/sa_ops.h.

The reference's training graph clips every tower's gradients to a global norm of 5 (lib/core/trainer.py:120-155); the names,
the argument order and the results follow the TensorFlow functions it calls.  The gradients may be of different types
(float32, bfloat16, float16); None entries are passed over.
"""
import ctypes
import functools
import operator

import torch

from .. import _tensor as T
from ... import _native as N

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_DTYPES = set(TYPES)
_dtype_of, _shape_of = operator.attrgetter("dtype"), operator.attrgetter("shape")
_device_of, _address_of = torch.Tensor.get_device, torch.Tensor.data_ptr


def _check(t, name):
    T.require(isinstance(t, torch.Tensor), "%s must be a torch.Tensor" % name)
    T.require(t.is_cuda, "%s must live on the GPU (the HIP path has no CPU fallback)" % name)
    T._on_current_device(t, name)
    T.require(t.dtype in TYPES, "%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))


def _dense_memory(t):
    """Every element of one block of memory exactly once, in any order of dimensions (a transposed matrix passes)."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _gather(t_list, op):
    """The tensors of the list (None entries dropped) and the device they are on, checked."""
    T.require(isinstance(t_list, (list, tuple)), "%s expects a list of tensors" % op)
    ts = [t for t in t_list if t is not None]
    device = torch.cuda.current_device() if torch.cuda.is_initialized() or torch.cuda.is_available() else -1
    # (maps over the methods: the host's share of a call on fifty small tensors is most of its time)
    if (device < 0 or not all([isinstance(t, torch.Tensor) for t in ts]) or not set(map(_device_of, ts)) <= {device}
            or not set(map(_dtype_of, ts)) <= _DTYPES):
        for i, t in enumerate(t_list):                 # say which
            if t is not None:
                _check(t, "t_list[%d]" % i)
        raise ValueError("%s needs a GPU (the HIP path has no CPU fallback)" % op)
    return ts, device


def _arrays(ts):
    k = len(ts)
    return ((ctypes.c_void_p * k)(*map(_address_of, ts)), (ctypes.c_long * k)(*map(torch.Tensor.numel, ts)),
            (ctypes.c_int * k)(*map(TYPES.__getitem__, map(_dtype_of, ts))))


@functools.lru_cache(maxsize=4096)
def _ws_bytes(count):
    n = ctypes.c_ulong()
    N.check(N.lib().sa_global_norm_ws(count, ctypes.byref(n)), "global_norm")
    return n.value


def _scalar_and_scratch(count, device):
    """The norm's fp32 scalar and the scratch of a call on `count` tensors."""
    size = _ws_bytes(count)
    return (torch.empty((), dtype=torch.float32, device=device), torch.empty(size, dtype=torch.uint8, device=device), size)


def _all_dense(ts):
    return all(map(torch.Tensor.is_contiguous, ts)) or all(map(_dense_memory, ts))


def _packed(ts):
    return ts if _all_dense(ts) else [t if _dense_memory(t) else t.contiguous() for t in ts]


def global_norm(t_list):
    """sqrt of the sum of all squares, a float32 scalar tensor on the GPU.  Sums are held in 64 bits, in a fixed order."""
    ts, device = _gather(t_list, "GlobalNorm")
    ts = _packed(ts)
    p, n, kinds = _arrays(ts)
    norm, ws, size = _scalar_and_scratch(len(ts), device)
    N.check(N.lib().sa_global_norm(len(ts), p, n, kinds, norm.data_ptr(), ws.data_ptr(), size,
                                   torch._C._cuda_getCurrentRawStream(device)), "global_norm")
    return norm


def _check_results(ts, results):
    for i, (t, o) in enumerate(zip(ts, results)):
        _check(o, "out[%d]" % i)
        T.require(o.shape == t.shape and o.dtype == t.dtype, "out[%d] differs from its gradient in shape or type" % i)
        # (the stride of a dimension of one element says nothing)
        T.require(t.numel() < 2 or all(a == b for a, b, n in zip(o.stride(), t.stride(), t.shape) if n != 1),
                  "out[%d] differs from its gradient in strides" % i)


def clip_by_global_norm(t_list, clip_norm, use_norm=None, out=None):
    """([t * clip_norm / max(norm, clip_norm) for t in t_list], norm).

    clip_norm: a positive number.  use_norm: a float32 scalar tensor on the GPU to use in place of the list's own norm (of
    gradients spread over several processes, say).  A norm that is NaN or infinite makes every result NaN, as in
    TensorFlow.  None entries stay None.

    out: None for new tensors, t_list itself to clip in place (nothing is written where the norm is within bounds), or a
    list of tensors of the same shapes and types.  Results must not overlap one another, nor any gradient but their own,
    which they may only share whole; each must be dense in memory, in its gradient's order of dimensions."""
    clip = float(clip_norm)
    T.require(clip > 0, "ClipByGlobalNorm expects a positive clip_norm")
    ts, device = _gather(t_list, "ClipByGlobalNorm")
    if use_norm is not None:
        _check(use_norm, "use_norm")
        T.require(use_norm.dtype == torch.float32 and use_norm.numel() == 1, "ClipByGlobalNorm expects a float32 scalar use_norm")
    if out is None:
        ts = _packed(ts)
        results = list(map(torch.empty_like, ts))
    else:
        T.require(isinstance(out, (list, tuple)) and len(out) == len(t_list), "ClipByGlobalNorm expects as many out tensors as gradients")
        if out is t_list:
            results = ts
        else:
            results = [o for o, t in zip(out, t_list) if t is not None]
            if not (all([isinstance(o, torch.Tensor) for o in results]) and set(map(_device_of, results)) <= {device} and
                    all(list(map(f, ts)) == list(map(f, results)) for f in (_shape_of, _dtype_of, torch.Tensor.stride))):
                _check_results(ts, results)
        T.require(_all_dense(ts), "a gradient that is not dense in memory cannot be clipped into out")
    p, n, kinds = _arrays(ts)
    o = (ctypes.c_void_p * len(ts))(*map(_address_of, results))
    if use_norm is None:
        norm, ws, size = _scalar_and_scratch(len(ts), device)
        given, to, scratch = None, norm.data_ptr(), ws.data_ptr()
    else:
        norm, size = use_norm, 0
        given, to, scratch = norm.data_ptr(), None, None
    N.check(N.lib().sa_clip_by_global_norm(len(ts), p, o, n, kinds, clip, given, to, scratch, size,
                                           torch._C._cuda_getCurrentRawStream(device)), "clip_by_global_norm")
    if len(results) == len(t_list):
        return results, norm
    it = iter(results)
    return [None if t is None else next(it) for t in t_list], norm
