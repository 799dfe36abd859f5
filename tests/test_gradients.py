"""tf_ops/gradients: the global norm of a list of gradients and clipping by it, against sums in 64 bits.

Bounds: the norm is a 64-bit sum rounded to fp32 (half a step, u = 2^-24, and as much again for the square root's own
rounding in 64 bits, which is far below).  A clipped value is g times a factor that carries two roundings (the norm's and its
own), multiplied in fp32 (one more) and rounded to its type (half a step h): (h + 4 u) |value|."""
import ctypes
import math

import pytest
import torch

from conftest import pkg

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _mod():
    return pkg("utils.tf_ops.gradients.tf_gradients")


def _rand(gpu, shape, dt=F32, seed=0, scale=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=gpu) * scale).to(dt)


def _norm64(ts):
    return math.sqrt(math.fsum(float(t.double().pow(2).sum()) for t in ts if t is not None))


def _check(ts, clip, got, norm, ref=None):
    ref = _norm64(ts) if ref is None else ref
    assert norm.dtype == F32 and norm.shape == () and abs(float(norm) - ref) <= 2 * U * ref
    f = min(1.0, clip / ref) if ref else 1.0
    assert len(got) == len(ts)
    for t, o in zip(ts, got):
        if t is None:
            assert o is None
            continue
        assert o.dtype == t.dtype and o.shape == t.shape
        want = t.double() * f
        info = torch.finfo(t.dtype)
        bound = (info.eps / 2 + 4 * U) * want.abs() + info.smallest_normal * info.eps
        assert bool(((o.double() - want).abs() <= bound).all())
        if f == 1.0:
            assert torch.equal(o, t)


LISTS = {
    "one element": [((1,), F32)],
    "one matrix": [((257, 129), BF16)],
    "mixed": [((64, 64), F32), ((1,), F16), ((3, 5, 7), BF16), ((100003,), F16), ((33,), F32), ((16384,), BF16), ((8192,), F32)],
    "chunk edges": [((n,), dt) for dt in (F32, BF16, F16) for n in (8191, 8192, 8193, 16383, 16384, 16385, 32769)],
    "empty among them": [((0,), F32), ((5,), F32), ((0, 3), BF16), ((7,), F16)],
    "128": [((i % 37 + 1,), F32) for i in range(128)],
    "129": [((i % 37 + 1,), (F32, BF16, F16)[i % 3]) for i in range(129)],
    "700": [((i * 7 % 5001 + 1,), (F32, BF16, F16)[i % 3]) for i in range(700)],
    "one large": [((40000001,), BF16)],
}


# ------------------------------------------------------------------------------------------------------- CPU: refusals
def test_refusals_without_a_gpu():
    m = _mod()
    with pytest.raises(ValueError, match="no CPU fallback"):
        m.global_norm([torch.zeros(3)])
    with pytest.raises(ValueError, match="list of tensors"):
        m.global_norm(torch.zeros(3))
    for bad in (0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="positive clip_norm"):
            m.clip_by_global_norm([], bad)
    with pytest.raises(ValueError, match="torch.Tensor"):
        m.clip_by_global_norm([3.0], 1.0)


def test_the_c_entries_refuse_bad_lists():
    lib = pkg("utils._native").lib()
    n = ctypes.c_ulong()
    assert lib.sa_global_norm_ws(-1, ctypes.byref(n)) == -1 and lib.sa_global_norm_ws(1, None) == -1
    assert lib.sa_global_norm_ws(0, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.sa_global_norm_ws(129, ctypes.byref(n)) == 0
    two = n.value
    assert lib.sa_global_norm_ws(128, ctypes.byref(n)) == 0 and two == 2 * n.value
    if torch.cuda.is_available():
        pytest.skip("made-up addresses below: only where nothing could be launched on them")
    a = 1 << 20                                        # never dereferenced: every call below is refused
    ptr, num, typ = (ctypes.c_void_p * 1)(a), (ctypes.c_long * 1)(5), (ctypes.c_int * 1)(0)
    assert lib.sa_global_norm(1, ptr, num, typ, a, None, 0, None) == -1                       # no scratch
    assert lib.sa_global_norm(1, ptr, num, typ, None, a, n.value, None) == -1                 # no result
    assert lib.sa_global_norm(1, None, num, typ, a, a, n.value, None) == -1
    assert lib.sa_global_norm(1, ptr, (ctypes.c_long * 1)(-5), typ, a, a, n.value, None) == -1
    assert lib.sa_global_norm(1, ptr, num, (ctypes.c_int * 1)(3), a, a, n.value, None) == -1
    assert lib.sa_global_norm(1, (ctypes.c_void_p * 1)(a + 2), num, typ, a, a, n.value, None) == -1   # half an element off
    assert lib.sa_clip_by_global_norm(1, ptr, ptr, num, typ, 0.0, None, a, a, n.value, None) == -1
    assert lib.sa_clip_by_global_norm(1, ptr, ptr, num, typ, float("nan"), None, a, a, n.value, None) == -1
    assert lib.sa_clip_by_global_norm(1, ptr, None, num, typ, 1.0, None, a, a, n.value, None) == -1
    assert lib.sa_clip_by_global_norm(1, ptr, ptr, num, typ, 1.0, None, None, a, n.value, None) == -1
    assert lib.sa_clip_by_global_norm(1, ptr, ptr, num, typ, 1.0, None, a, a, n.value - 1, None) == -1
    # results that overlap one another, another gradient, or the norm that is read; scratch of a later check missing
    def pair(p0, p1, o0, o1, n0, n1, use=None):
        return lib.sa_clip_by_global_norm(2, (ctypes.c_void_p * 2)(p0, p1), (ctypes.c_void_p * 2)(o0, o1), (ctypes.c_long * 2)(n0, n1),
                                          (ctypes.c_int * 2)(0, 0), 1.0, use, None, None, 0, None)
    assert pair(a, a + 400, a, a + 396, 100, 100) == -1 and pair(a, a, a, a, 100, 100) == -1
    assert pair(a, a, a, a + 4000, 100, 100) == -1 and pair(a, a + 400, a + 400, a, 100, 100) == -1
    assert pair(a, a + 400, a + 4, a + 8000, 100, 100) == -1 and pair(a, a + 400, a, a + 400, 100, 100, a + 796) == -1


# --------------------------------------------------------------------------------------------------------- GPU: values
@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(LISTS))
def test_lists_of_every_kind(gpu, name):
    m = _mod()
    ts = [_rand(gpu, s, dt, i, 10.0 ** (i % 3 - 1)) for i, (s, dt) in enumerate(LISTS[name])]
    ref = _norm64(ts)
    norm = m.global_norm(ts)
    assert abs(float(norm) - ref) <= 2 * U * ref and torch.equal(m.global_norm(ts), norm)
    for clip in (ref / 3, ref * 3):
        got, n = m.clip_by_global_norm(ts, clip)
        assert torch.equal(n, norm)
        _check(ts, clip, got, n, ref)
        mine = [t.clone() for t in ts]
        same, n = m.clip_by_global_norm(mine, clip, out=mine)
        assert all(a is b for a, b in zip(same, mine)) and torch.equal(n, norm)
        assert all(torch.equal(a, b) for a, b in zip(mine, got))
        into = [torch.full_like(t, 3.0) for t in ts]
        m.clip_by_global_norm(ts, clip, use_norm=norm, out=into)
        assert all(torch.equal(a, b) for a, b in zip(into, got))


@pytest.mark.gpu
def test_nothing_to_clip(gpu):
    m = _mod()
    for ts in ([], [None], [None, torch.empty(0, device=gpu)]):
        got, norm = m.clip_by_global_norm(ts, 1.0)
        assert float(norm) == 0.0 and len(got) == len(ts) and got[0] is None if ts else got == []
        assert float(m.global_norm(ts)) == 0.0
    zero = [torch.zeros(100, device=gpu), None]
    got, norm = m.clip_by_global_norm(zero, 1.0)
    assert float(norm) == 0.0 and torch.equal(got[0], zero[0]) and got[1] is None
    t = [_rand(gpu, (1000,))]
    got, norm = m.clip_by_global_norm(t, float("inf"))
    assert torch.equal(got[0], t[0])


@pytest.mark.gpu
def test_views_unaligned_and_in_any_order_of_dimensions(gpu):
    m = _mod()
    for dt in (F32, BF16, F16):
        for off in (1, 3, 5):
            flat = _rand(gpu, (100 + 50000,), dt, off)
            guard = flat.clone()
            ts = [flat[off:off + 40001], flat[off + 40001:off + 40010]]      # neighbours in one buffer
            ref = _norm64(ts)
            _check(ts, ref / 2, *m.clip_by_global_norm(ts, ref / 2))
            shifted = [torch.full((40012,), 9.0, dtype=dt, device=gpu) for _ in ts]
            into = [s[2:2 + t.numel()] for s, t in zip(shifted, ts)]         # results aligned unlike their gradients
            _check(ts, ref / 2, *m.clip_by_global_norm(ts, ref / 2, out=into))
            for s, t in zip(shifted, ts):
                assert bool((s[:2] == 9).all()) and bool((s[2 + t.numel():] == 9).all())
            want, _ = m.clip_by_global_norm(ts, ref / 2)
            m.clip_by_global_norm(ts, ref / 2, out=ts)
            assert all(torch.equal(a, b) for a, b in zip(ts, want))
            assert torch.equal(flat[:off], guard[:off]) and torch.equal(flat[off + 40010:], guard[off + 40010:])
        mat = _rand(gpu, (65, 33), dt, 7)
        ts = [mat.t(), _rand(gpu, (4, 6, 10), dt, 8).permute(2, 0, 1), _rand(gpu, (20, 9), dt, 9)[:, :4]]
        ref = _norm64(ts)
        got, norm = m.clip_by_global_norm(ts, ref / 2)
        _check(ts, ref / 2, got, norm)
        want = got[0].clone()
        m.clip_by_global_norm(ts[:2], 1.0, use_norm=norm * (2 / ref), out=ts[:2])
        assert want.shape == ts[0].shape


@pytest.mark.gpu
def test_large_and_small_values_and_those_that_are_no_numbers(gpu):
    m = _mod()
    for v in (1e25, 1e-25, 1e-38):                     # squares beyond fp32's range at both ends
        ts = [torch.full((5000,), v, device=gpu), torch.full((3,), v, device=gpu).to(BF16)]
        ref = _norm64(ts)
        _check(ts, ref / 4, *m.clip_by_global_norm(ts, ref / 4))
    for bad in (float("nan"), float("inf"), -float("inf")):
        ts = [_rand(gpu, (4000,), F32, 1), _rand(gpu, (50,), F16, 2), _rand(gpu, (0,), BF16, 3)]
        ts[0][1234] = bad
        for kw in ({}, {"out": [t.clone() for t in ts]}):
            got, norm = m.clip_by_global_norm(ts, 1.0, **kw)
            assert not math.isfinite(float(norm)) and all(bool(torch.isnan(g).all()) for g in got)
        m.clip_by_global_norm(ts, 1.0, out=ts)
        assert all(bool(torch.isnan(t).all()) for t in ts)


@pytest.mark.gpu
def test_streams_and_graphs(gpu):
    m = _mod()
    ts = [_rand(gpu, (4097 * (i + 1),), (F32, BF16, F16)[i % 3], i) for i in range(20)]
    want, norm = m.clip_by_global_norm(ts, 5.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, n2 = m.clip_by_global_norm(ts, 5.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(want, other))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m.clip_by_global_norm(ts, 5.0)
        graphs.append((g, out))
    for turn in range(3):
        for i, t in enumerate(ts):
            t.copy_(_rand(gpu, t.shape, t.dtype, 100 * turn + i, 10.0 ** -turn))
        eager, norm = m.clip_by_global_norm(ts, 5.0)
        for g, (got, n2) in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(got, eager))


@pytest.mark.gpu
def test_refused_lists(gpu):
    m = _mod()
    a, b = torch.ones(10, device=gpu), torch.ones(10, device=gpu)
    for ts, kw in (([a, a], dict(out="same")), ([a[:6], a[4:]], dict(out="same")), ([a], dict(out=[])),
                   ([a], dict(out=[b.half()])), ([a], dict(out=[b[:9]])), ([a], dict(out=[torch.ones(20, device=gpu)[::2]])),
                   ([a, b], dict(out=[b, a])), ([a[:8], b], dict(out=[a[2:], b])), ([a.double()], {}), ([a.int()], {}),
                   ([a], dict(use_norm=torch.ones(2, device=gpu))), ([a], dict(use_norm=torch.ones(()))),
                   ([a], dict(use_norm=a[3], out=[a])), ([torch.ones(20, device=gpu)[::2]], dict(out="same")),
                   ([torch.ones(1, device=gpu).expand(5)], dict(out="same"))):
        if kw.get("out") == "same":
            kw = dict(out=ts)
        with pytest.raises(ValueError):
            m.clip_by_global_norm(ts, 1.0, **kw)
    got, norm = m.clip_by_global_norm([a, a], 1.0)      # the same gradient twice counts twice
    _check([a, a], 1.0, got, norm)


@pytest.mark.gpu
def test_a_tensor_of_more_than_32_bits_of_elements(gpu):
    m = _mod()
    t = torch.zeros((1 << 31) + 77, dtype=torch.bfloat16, device=gpu)
    t[:2], t[-3:] = 3.0, 4.0
    assert abs(float(m.global_norm([t])) - 66.0 ** 0.5) <= 2.0 ** -23 * 66.0 ** 0.5
    m.clip_by_global_norm([t], 1.0, out=[t])
    # one division of 64 bits, two roundings to fp32 and one to bf16
    assert all(abs(float(v) - want / 66.0 ** 0.5) <= 2.0 ** -7.9 * want / 66.0 ** 0.5 for v, want in ((t[0], 3.0), (t[-1], 4.0)))
    assert int((t != 0).sum()) == 5


@pytest.mark.gpu
def test_factors_below_the_normal_range(gpu):
    """clip / norm may be as small as 1e-46 / 1e38 while the clipped values are ordinary numbers."""
    m = _mod()
    for v, clip in ((1e36, 1e-3), (1e36, 1e-9), (1e35, 1e-20), (3e36, 3.0), (3e33, 1e-5), (3e37, 5.0)):
        ts = [torch.full((40,), v, device=gpu), torch.full((3,), -v / 3, device=gpu).to(BF16), _rand(gpu, (77,), F32, 1, v / 10),
              _rand(gpu, (9,), F16, 2)]
        into = [torch.full((t.numel() + 1,), 9.0, dtype=t.dtype, device=gpu)[1:] for t in ts]     # aligned unlike the gradients
        mine = [t.clone() for t in ts]
        for kw in ({}, {"out": into}, {"out": mine}):
            src = mine if "out" in kw and kw["out"] is mine else ts
            got, norm = m.clip_by_global_norm(src, clip, **kw)
            _check(ts, clip, got, norm)
    big = [torch.full((20000,), 1e35, device=gpu)]     # whole chunks too
    _check(big, 1e-8, *m.clip_by_global_norm(big, 1e-8))
