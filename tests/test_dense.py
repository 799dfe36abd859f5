"""tf_ops/dense: the dense layer with its epilogue, and its gradient, against the formulas in 64 bits.

Bounds, per element.  u = 2^-24 is half a step of fp32, h = eps / 2 half a step of the layer's type.  A sum of K products
computed in fp32 in any order is off by about sqrt(K) u times S = sum |x||w| (rounding errors of random sign; 8 sqrt(K) is
eight standard deviations), plus a few u for what happens to the sum afterwards: bias, activation (Lipschitz constant < 1.2,
exp and erfc within a few u of values no larger than |z| + 1), residual.  The result is rounded once: h |y|.  In the
gradient the 16-bit types round dz once (h |dz| per factor), which passes through the products with |w| and |x|."""
import ctypes
import math

import pytest
import torch

from conftest import pkg

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def _mod():
    return pkg("utils.tf_ops.dense.tf_dense")


def _half(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps       # half steps below the normal range


def _act64(z, act):
    if act is None:
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z)


def _slope64(z, act):
    if act is None:
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def _sum_bound(k):
    return (8 * math.sqrt(max(k, 1)) + 16) * U


def _within(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), "%s: %d of %d outside, worst %.3g of its bound at %s" % (
        what, int(bad.sum()), bad.numel(), float((err / bound).max()), bad.nonzero()[0].tolist())


def _check_forward(x, w, b, act, res, out, pre):
    dt = x.dtype
    xd, wd = x.double(), w.double()
    z = xd @ wd.contiguous()
    s = xd.abs() @ wd.abs().contiguous()
    if b is not None:
        z, s = z + b.double(), s + b.double().abs()
    dz = _sum_bound(w.shape[0]) * s + 4 * U * z.abs()
    if pre is not None:
        _within(pre, z, _half(dt) * (z.abs() + dz) + dz + _tiny(dt), "preact")
    y = _act64(z, act)
    bound = 1.2 * dz + 16 * U * (z.abs() + 1) * (act not in (None, "relu"))
    if res is not None:
        y = y + res.double()
        bound = bound + 2 * U * (y.abs() + res.double().abs())
    _within(out, y, _half(dt) * (y.abs() + bound) + bound + _tiny(dt), "out")


def _check_grad(x, w, g, act, z, dx, dw, db):
    dt = x.dtype
    gd = g.double()
    d = gd if act is None else gd * _slope64(z.double(), act)
    # slope: a few steps of terms no larger than 1.2 (1 + |z|); one rounding to the type where there is an activation
    dd = 0 * d if act is None else 32 * U * gd.abs() * (1 + z.double().abs()) + _tiny(torch.float32)
    dr = dd if act is None or dt == torch.float32 else dd + _half(dt) * (d.abs() + dd) + _tiny(dt)
    xd, wd = x.double(), w.double()
    if dx is not None:
        want = d @ wd.t().contiguous()
        b = (_sum_bound(w.shape[1]) * (d.abs() + dr) + dr) @ wd.abs().t().contiguous()
        _within(dx, want, _half(dt) * (want.abs() + b) + b + _tiny(dt), "grad_inputs")
    if dw is not None:
        xt = xd.t().contiguous()
        want = xt @ d
        b = xt.abs() @ (_sum_bound(x.shape[0]) * (d.abs() + dr) + dr)
        _within(dw, want, _half(dt) * (want.abs() + b) + b + _tiny(dt), "grad_weights")
    if db is not None:
        want = d.sum(0)
        b = (_sum_bound(x.shape[0]) * (d.abs() + dd) + dd).sum(0)
        _within(db, want, _half(db.dtype) * (want.abs() + b) + b + _tiny(db.dtype), "grad_biases")


def _rand(gpu, shape, dt, seed, scale=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=gpu) * scale).to(dt)


# (rows, cin, cout): one row to thousands, odd and aligned widths, one column, one channel, tiles' edges and one past them
SIZES = [(1, 1, 1), (1, 64, 8), (1, 1027, 515), (3, 5, 7), (17, 67, 33), (64, 64, 64), (65, 65, 65), (128, 256, 128),
         (129, 257, 130), (300, 131, 1), (5, 2048, 24), (33, 4096, 257), (1000, 96, 200), (257, 512, 384), (515, 771, 259),
         (2048, 512, 128), (1, 4096, 1024), (8, 1024, 1000), (16, 640, 512), (31, 1000, 2048), (4099, 40, 72),
         # products of the tile kernel: its edges, odd operands (copied first), many and few tiles, short and long k
         (640, 520, 648), (33, 8192, 520), (129, 1030, 2056), (3585, 72, 3400), (2049, 2065, 33), (70001, 40, 33), (384, 4096, 256),
         (4100, 72, 4104), (8200, 136, 1032), (1100, 1100, 1100), (30001, 264, 520), (520, 30001, 136), (2050, 1027, 1030),
         # narrow on one side: products of few steps, with and without a bias in them
         (7, 3217, 1603), (24, 1862, 1394), (12501, 265, 8), (16389, 8, 517), (65, 2051, 1112), (64, 2048, 1153)]


# ------------------------------------------------------------------------------------------------------- CPU: refusals
def test_cpu_tensors_and_unknown_activations_are_refused():
    m = _mod()
    x, w = torch.zeros(2, 3), torch.zeros(3, 4)
    with pytest.raises(ValueError, match="no CPU fallback"):
        m.dense(x, w)
    with pytest.raises(ValueError, match="no CPU fallback"):
        m.dense_grad(x, w, torch.zeros(2, 4))
    with pytest.raises(ValueError, match="torch.Tensor"):
        m.dense(None, w)


def test_the_c_entries_refuse_what_they_cannot_compute():
    lib = pkg("utils._native").lib()
    n = ctypes.c_ulong()
    by = ctypes.byref(n)
    assert lib.sa_dense_forward_ws(3, 1, 1, 1, 0, by) == -1 and lib.sa_dense_forward_ws(0, -1, 1, 1, 0, by) == -1
    assert lib.sa_dense_forward_ws(0, 1, 1 << 24, 1, 0, by) == -1
    assert lib.sa_dense_forward_ws(0, 1, 1, 1, 0, None) == -1
    assert lib.sa_dense_backward_ws(0, 1, 1, 1, 9, 7, 0, by) == -1 and lib.sa_dense_backward_ws(0, 1, 1, 1, 0, 8, 0, by) == -1
    if torch.cuda.is_available():
        pytest.skip("made-up addresses below: only where nothing could be launched on them")
    p = 1 << 20                                        # an address that is never dereferenced: every call below is refused
    fwd = lambda **k: lib.sa_dense_forward(*[k.get(a, d) for a, d in (   # noqa: E731
        ("dtype", 1), ("rows", 4), ("cin", 8), ("cout", 8), ("x", p), ("ldx", 8), ("w", p), ("ldw", 8), ("bias", None), ("bf", 0),
        ("res", None), ("ldr", 0), ("act", 0), ("y", p), ("pre", None), ("ws", None), ("wsb", 0), ("stream", None))])
    assert fwd(dtype=7) == -1 and fwd(act=5) == -1 and fwd(act=-1) == -1 and fwd(rows=-1) == -1
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(y=None) == -1
    assert fwd(ldx=7) == -1 and fwd(ldw=7) == -1 and fwd(res=p, ldr=7) == -1
    assert fwd(rows=0) == 0 and fwd(cout=0) == 0       # nothing to compute
    assert lib.sa_dense_forward_ws(1, 400, 4096, 8, 3, by) == 0 and n.value > 0
    assert fwd(rows=400, cin=4096, ldx=4096) == -1     # scratch missing
    assert fwd(rows=400, cin=4096, ldx=4096, ws=p, wsb=n.value - 1) == -1
    assert fwd(ldx=1 << 24) == -3 and fwd(ldw=1 << 24) == -3   # offsets inside a tile would not fit
    bwd = lambda **k: lib.sa_dense_backward(*[k.get(a, d) for a, d in (   # noqa: E731
        ("dtype", 1), ("rows", 4), ("cin", 8), ("cout", 8), ("x", p), ("ldx", 8), ("w", p), ("ldw", 8), ("g", p), ("ldg", 8),
        ("z", p), ("ldz", 8), ("act", 1), ("dx", p), ("dw", p), ("db", p), ("df", 0), ("ws", None), ("wsb", 0), ("stream", None))])
    assert lib.sa_dense_backward_ws(1, 4000, 1000, 1000, 1, 7, 7, by) == 0 and n.value > 0
    wide = dict(rows=4000, cin=1000, cout=1000, ldx=1000, ldw=1000, ldg=1000, ldz=1000)
    assert bwd(**wide) == -1 and bwd(ws=p, wsb=n.value - 1, **wide) == -1      # scratch missing, scratch too small
    assert bwd(g=None) == -1 and bwd(z=None) == -1 and bwd(x=None) == -1 and bwd(w=None) == -1 and bwd(ldg=7) == -1
    assert bwd(dx=None, dw=None, db=None) == 0 and bwd(ldg=1 << 24) == -3 and bwd(ldw=1 << 24) == -3


# --------------------------------------------------------------------------------------------------------- GPU: values
@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_dense_matches_64_bits(gpu, size, dt):
    m = _mod()
    rows, cin, cout = size
    i = SIZES.index(size)
    x, w = _rand(gpu, (rows, cin), dt, i), _rand(gpu, (cin, cout), dt, 100 + i, math.sqrt(2.0 / cin))
    b = _rand(gpu, (cout,), torch.float32 if i % 2 else dt, 200 + i)
    res = _rand(gpu, (rows, cout), dt, 300 + i)
    act = ACTS[i % 5]
    out, pre = m.dense(x, w, b, activation=act, residual=res, return_preact=True)
    assert out.dtype == dt and out.shape == (rows, cout) and pre.shape == out.shape
    _check_forward(x, w, b, act, res, out, pre)
    plain = m.dense(x, w)
    _check_forward(x, w, None, None, None, plain, None)
    assert torch.equal(m.dense(x, w), plain)           # the same call, the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 1, 4])
@pytest.mark.parametrize("size", [(600, 1020, 1604), (1031, 1021, 1027), (32773, 44, 700), (7000, 68, 2100), (150, 6004, 1029),
                                  (66000, 96, 256), (8192, 2052, 68), (16400, 1028, 72), (9000, 2600, 300)])
def test_large_fp32_products_at_odd_places(gpu, size, pad):
    """Lengths that end inside a step of 32, rows 16-byte aligned and not, kept sums, a residual, and none."""
    m = _mod()
    rows, cin, cout = size
    i = rows + pad
    big = _rand(gpu, (rows, cin + pad), torch.float32, i)
    big[:, :pad] = float("nan")
    x, w = big[:, pad:], _rand(gpu, (cin, cout), torch.float32, i + 1, math.sqrt(2.0 / cin))
    b, res = _rand(gpu, (cout,), torch.float32, i + 2), _rand(gpu, (rows, cout), torch.float32, i + 3)
    out, pre = m.dense(x, w, b, activation="silu", residual=res, return_preact=True)
    _check_forward(x, w, b, "silu", res, out, pre)
    plain = m.dense(x, w)
    _check_forward(x, w, None, None, None, plain, None)
    assert torch.equal(m.dense(x, w), plain)
    g = _rand(gpu, (rows, cout), torch.float32, i + 4, 0.05)
    for act in ("silu", None):
        dx, dw, db = m.dense_grad(x, w, g, biases=b, activation=act, preact=pre if act else None)
        _check_grad(x, w, g, act, pre, dx, dw, db)
        assert torch.equal(m.dense_grad(x, w, g, activation=act, preact=pre, needs=(False, True))[1], dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_every_activation_over_its_whole_range(gpu, act, dt):
    # one channel in, weight 1: z is the input itself, from the tails to zero
    m = _mod()
    x = torch.cat([torch.linspace(-40, 40, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e4, -1e4])]).to(gpu).to(dt)[:, None]
    w = torch.ones(1, 1, dtype=dt, device=gpu)
    out, pre = m.dense(x, w, activation=act, return_preact=True)
    assert torch.equal(pre, x + 0)
    _check_forward(x, w, None, act, None, out, pre)
    g = torch.ones_like(x)
    dx, dw, db = m.dense_grad(x, w, g, biases=torch.zeros(1, dtype=dt, device=gpu), activation=act, preact=pre)
    _check_grad(x, w, g, act, pre, dx, dw, None)       # (4 007 terms of which all but a few are small: see the sums' test)
    assert torch.isfinite(out).all() and torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_dense_grad_matches_64_bits(gpu, size, dt):
    m = _mod()
    rows, cin, cout = size
    i = SIZES.index(size)
    act = ACTS[(i + 2) % 5]
    x, w = _rand(gpu, (rows, cin), dt, i), _rand(gpu, (cin, cout), dt, 100 + i, math.sqrt(2.0 / cin))
    g, z = _rand(gpu, (rows, cout), dt, 200 + i, 0.05), _rand(gpu, (rows, cout), dt, 300 + i)
    b = torch.empty(cout, dtype=torch.float32 if i % 2 else dt, device=gpu)
    dx, dw, db = m.dense_grad(x, w, g, biases=b, activation=act, preact=z)
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape and db.dtype == b.dtype
    _check_grad(x, w, g, act, z, dx, dw, db)
    only_x = m.dense_grad(x, w, g, activation=act, preact=z, needs=(True, False))
    only_w = m.dense_grad(x, w, g, activation=act, preact=z, needs=(False, True))
    assert only_x[1] is None and only_x[2] is None and torch.equal(only_x[0], dx)
    assert only_w[0] is None and torch.equal(only_w[1], dw)


@pytest.mark.gpu
def test_dense_grad_against_differences(gpu):
    # phi(t) = <g, dense(x + t dx, w + t dw, b + t db)> has the slope that the gradients give; central differences in fp32:
    # error h^2 / 6 phi''' ~ 1e-4 of the terms' size plus the rounding of phi, u |phi| / h ~ 1e-4
    m = _mod()
    rows, cin, cout = 37, 61, 45
    for k, act in enumerate(["gelu", "gelu_tanh", "silu", None]):
        x, w, b = _rand(gpu, (rows, cin), torch.float32, k), _rand(gpu, (cin, cout), torch.float32, 10 + k, 0.15), _rand(
            gpu, (cout,), torch.float32, 20 + k)
        g = _rand(gpu, (rows, cout), torch.float32, 30 + k)
        vx, vw, vb = (_rand(gpu, t.shape, torch.float32, 40 + k + i, 0.1) for i, t in enumerate((x, w, b)))
        h = 1e-2
        phi = [float((m.dense(x + s * h * vx, w + s * h * vw, b + s * h * vb, activation=act).double() * g.double()).sum())
               for s in (1, -1)]
        _, z = m.dense(x, w, b, activation=act, return_preact=True)
        dx, dw, db = m.dense_grad(x, w, g, biases=b, activation=act, preact=z)
        slope = sum(float((a.double() * v.double()).sum()) for a, v in ((dx, vx), (dw, vw), (db, vb)))
        size = math.sqrt(sum(float((a.double() * v.double()).pow(2).sum()) for a, v in ((dx, vx), (dw, vw), (db, vb))))
        assert abs((phi[0] - phi[1]) / (2 * h) - slope) < 2e-3 * max(size, abs(slope)), act


# ---------------------------------------------------------------------------------------- GPU: layouts, edges, neighbours
@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_strides_offsets_and_leading_dimensions(gpu, dt):
    m = _mod()
    nan = float("nan")
    for cin, cout, pad in ((64, 72, 8), (67, 33, 5), (512, 256, 64), (131, 515, 1)):
        rows = 150
        big_x, big_w = torch.full((rows, cin + pad), nan, dtype=dt, device=gpu), torch.full((cin, cout + pad), nan, dtype=dt, device=gpu)
        big_r, big_g = (torch.full((rows, cout + pad), nan, dtype=dt, device=gpu) for _ in range(2))
        x, w, r, g = big_x[:, pad:], big_w[:, :cout], big_r[:, pad:], big_g[:, :cout]     # NaN between the rows
        x.copy_(_rand(gpu, x.shape, dt, 1)); w.copy_(_rand(gpu, w.shape, dt, 2, 0.1))     # noqa: E702
        r.copy_(_rand(gpu, r.shape, dt, 3)); g.copy_(_rand(gpu, g.shape, dt, 4))          # noqa: E702
        b = _rand(gpu, (2 * cout,), dt, 5)[::2]                                           # a strided bias
        out, pre = m.dense(x, w, b, activation="silu", residual=r, return_preact=True)
        _check_forward(x, w, b, "silu", r, out, pre)
        dx, dw, db = m.dense_grad(x, w, g, biases=b, activation="silu", preact=pre)
        _check_grad(x, w, g, "silu", pre, dx, dw, db)
        # a transposed weight, a column-major input, broadcast rows and residual
        wt = w.t().contiguous().t()
        xt = x.t().contiguous().t()
        assert not wt.is_contiguous() and not xt.is_contiguous()
        ref = m.dense(x.contiguous(), w.contiguous(), activation="relu")
        assert torch.equal(m.dense(xt, wt, activation="relu"), ref)
        one = x[:1].expand(rows, cin)
        _check_forward(one, w, None, None, r[:1].expand(rows, cout), m.dense(one, w, residual=r[:1].expand(rows, cout)), None)
        # more leading dimensions, and none
        x3 = x.contiguous().view(3, 50, cin)
        assert torch.equal(m.dense(x3, w.contiguous(), activation="relu"), ref.view(3, 50, cout))
        assert m.dense(x3[:, ::2], w).shape == (3, 25, cout)
        _check_forward(x3[:, ::2].reshape(-1, cin), w, None, None, None, m.dense(x3[:, ::2], w).view(-1, cout), None)
        v = m.dense(x[0], w)
        assert v.shape == (cout,)
        _check_forward(x[:1], w, None, None, None, v[None], None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_empty_sizes(gpu, dt):
    m = _mod()
    new = lambda *s: torch.randn(*s, device=gpu).to(dt)  # noqa: E731
    assert m.dense(new(0, 5), new(5, 7)).shape == (0, 7) and m.dense(new(3, 5), new(5, 0)).shape == (3, 0)
    b, r = new(7), new(3, 7)
    out = m.dense(new(3, 0), new(0, 7), b, activation="relu", residual=r)
    assert torch.equal(out, (torch.relu(b.float()) + r.float()).to(dt))
    dx, dw, db = m.dense_grad(new(0, 5), new(5, 7), new(0, 7), biases=b, activation="relu", preact=new(0, 7))
    assert dx.shape == (0, 5) and torch.equal(dw, torch.zeros(5, 7, dtype=dt, device=gpu)) and torch.equal(db, torch.zeros_like(b))
    dx, dw, db = m.dense_grad(new(3, 5), new(5, 0), new(3, 0), biases=new(0))
    assert torch.equal(dx, torch.zeros(3, 5, dtype=dt, device=gpu)) and dw.shape == (5, 0) and db.shape == (0,)
    dx, dw, db = m.dense_grad(new(3, 0), new(0, 7), r, biases=b)
    assert dx.shape == (3, 0) and dw.shape == (0, 7)
    _within(db, r.double().sum(0), _half(dt) * r.double().sum(0).abs() + 8 * U * r.double().abs().sum(0), "grad_biases")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_infinities_and_nans_stay_in_their_rows_and_columns(gpu, dt):
    m = _mod()
    for rows, cin, cout in ((70, 129, 65), (512, 256, 512), (3, 512, 256)):
        x, w = _rand(gpu, (rows, cin), dt, 1), _rand(gpu, (cin, cout), dt, 2)
        clean = m.dense(x, w)
        x[1, 3] = float("nan")
        w[5, 7] = float("inf")
        out = m.dense(x, w)
        assert torch.isnan(out[1]).all()
        assert not torch.isfinite(out[:, 7]).any()
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1] = False
        keep[:, 7] = False
        assert torch.equal(out[keep], clean[keep])
        assert torch.isnan(m.dense(x, w, activation="relu")[1]).all()
    # what reaches a closed ReLU does not come through, infinities included
    z = torch.tensor([[-1.0, 0.0, 2.0, -3.0]], device=gpu).to(dt)
    g = torch.tensor([[float("inf"), float("nan"), 1.0, 2.0]], device=gpu).to(dt)
    x, w = torch.ones(1, 2, dtype=dt, device=gpu), torch.ones(2, 4, dtype=dt, device=gpu)
    dx, dw, db = m.dense_grad(x, w, g, biases=torch.zeros(4, dtype=dt, device=gpu), activation="relu", preact=z)
    assert db.tolist() == [0.0, 0.0, 1.0, 0.0] and dx.tolist() == [[1.0, 1.0]] and dw.tolist() == [[0.0, 0.0, 1.0, 0.0]] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [(3, 512, 256), (257, 131, 67), (1024, 1024, 1024), (1031, 1021, 1027), (33000, 128, 256)])
def test_infinities_have_the_sign_of_the_product(gpu, dt, size):
    """One infinite factor among finite ones gives an infinity of the product's sign, two of opposite signs and infinity times
    zero NaN -- also where the other factor has few bits (1) or many, is large or small.  (The exact sums are rounded to the
    type first: fp16 has no 86462.)"""
    m = _mod()
    rows, cin, cout = size
    inf = float("inf")
    x, w = _rand(gpu, (rows, cin), dt, 1), _rand(gpu, (cin, cout), dt, 2)
    w[3, :40:2], w[3, 1:41:2] = 1.0, -1.0                  # what the infinities below meet
    w[3, 41:50] = torch.tensor([0.0, 3e4, -3e4, 1.001, -1.001, 3e-5, -3e-5, 511.5, -511.5], device=gpu).to(dt)
    x[:, 5] = torch.where(x[:, 5] == 0, torch.ones((), dtype=dt, device=gpu), x[:, 5])
    x[2, 5] = 0.0
    x[1, 3], x[rows - 1, 3] = inf, -inf
    w[5, 7], w[5, 60] = -inf, inf
    x[rows // 2, 5] = inf                                  # meets the infinities of w
    out, expected = m.dense(x, w), (x.double() @ w.double()).to(dt)
    for ours, theirs in ((torch.isnan(out), torch.isnan(expected)), (out == inf, expected == inf), (out == -inf, expected == -inf)):
        assert torch.equal(ours, theirs)
    g = _rand(gpu, (rows, cout), dt, 3)
    g[1, 3], g[rows - 1, 5] = inf, -inf
    dx, dw, _ = m.dense_grad(x, w, g)
    for out, expected in ((dx, (g.double() @ w.double().T).to(dt)), (dw, (x.double().T @ g.double()).to(dt))):
        for ours, theirs in ((torch.isnan(out), torch.isnan(expected)), (out == inf, expected == inf), (out == -inf, expected == -inf)):
            assert torch.equal(ours, theirs)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [(5, 64, 40), (131, 67, 259), (300, 512, 264), (2048, 512, 128), (33003, 132, 259)])
def test_nothing_is_written_outside_the_outputs(gpu, dt, size):
    lib, m = pkg("utils._native").lib(), _mod()
    rows, cin, cout = size
    x, w, g, z = (_rand(gpu, s, dt, i) for i, s in enumerate(((rows, cin), (cin, cout), (rows, cout), (rows, cout))))
    code = m.TYPES[dt]
    guard = 4096

    def padded(n):
        t = torch.full((n + 2 * guard,), 7.0, dtype=dt, device=gpu)
        return t, t[guard:guard + n]

    def intact(t, n):
        return bool((t[:guard] == 7).all()) and bool((t[guard + n:] == 7).all())

    ws_all, st = {}, torch.cuda.current_stream().cuda_stream

    def scratch(need):
        t = torch.full((need + 8192,), 11, dtype=torch.uint8, device=gpu)
        ws_all[need] = t
        return t

    al = lambda *ts: sum(1 << i for i, t in enumerate(ts) if t.data_ptr() % 16 == 0 and t.shape[1] * t.element_size() % 16 == 0)  # noqa: E731
    n = ctypes.c_ulong()
    assert lib.sa_dense_forward_ws(code, rows, cin, cout, al(x, w), ctypes.byref(n)) == 0
    ws = scratch(n.value)
    (yb, y), (pb, p) = padded(rows * cout), padded(rows * cout)
    assert lib.sa_dense_forward(code, rows, cin, cout, x.data_ptr(), cin, w.data_ptr(), cout, None, 0, None, 0, 4, y.data_ptr(),
                                p.data_ptr(), ws.data_ptr(), n.value, st) == 0
    assert intact(yb, rows * cout) and intact(pb, rows * cout) and bool((ws[n.value:] == 11).all())
    assert torch.equal(y.view(rows, cout), m.dense(x, w, activation="silu"))
    assert lib.sa_dense_backward_ws(code, rows, cin, cout, 4, 7, al(x, w, g), ctypes.byref(n)) == 0
    ws = scratch(n.value)
    (xb, dx), (wb, dw), (bb, db) = padded(rows * cin), padded(cin * cout), padded(cout)
    assert lib.sa_dense_backward(code, rows, cin, cout, x.data_ptr(), cin, w.data_ptr(), cout, g.data_ptr(), cout, z.data_ptr(),
                                 cout, 4, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), 0, ws.data_ptr(), n.value, st) == 0
    assert intact(xb, rows * cin) and intact(wb, cin * cout) and intact(bb, cout) and bool((ws[n.value:] == 11).all())


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    # 2^26 + 70 rows of 40 channels: element offsets pass 2^31, byte offsets 2^32
    m = _mod()
    rows, cin, cout = (1 << 26) + 70, 40, 8
    x = torch.zeros(rows, cin, dtype=torch.bfloat16, device=gpu)
    w = _rand(gpu, (cin, cout), torch.bfloat16, 1)
    x[-100:] = _rand(gpu, (100, cin), torch.bfloat16, 2)
    out = m.dense(x, w)
    _check_forward(x[-100:], w, None, None, None, out[-100:], None)
    assert not bool(out[:-100].any())
    _, dw, _ = m.dense_grad(x, w, out, needs=(False, True))
    _check_grad(x[-100:], w, out[-100:], None, None, None, dw, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,cin,cout", [(torch.float32, 1100, 40), (torch.bfloat16, 2200, 40), (torch.bfloat16, 40, 2200)])
def test_large_products_with_offsets_past_32_bits(gpu, dt, cin, cout):
    m = _mod()
    rows = (1 << 20) + 70                              # inputs, or results, of more than 2^32 bytes
    x, g = torch.zeros(rows, cin, dtype=dt, device=gpu), torch.zeros(rows, cout, dtype=dt, device=gpu)
    w = _rand(gpu, (cin, cout), dt, 1, 0.05)
    x[-100:], g[-100:] = _rand(gpu, (100, cin), dt, 2), _rand(gpu, (100, cout), dt, 3)
    out = m.dense(x, w)
    _check_forward(x[-100:], w, None, None, None, out[-100:], None)
    assert not bool(out[:-100].any())
    del out
    dx, dw, _ = m.dense_grad(x, w, g)
    assert not bool(dx[:-100].any())
    _check_grad(x[-100:], w, g[-100:], None, None, dx[-100:], dw, None)


# ------------------------------------------------------------------------------------------- GPU: streams, graphs, refusals
@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_other_streams_and_captured_graphs_give_the_same_bits(gpu, dt):
    m = _mod()
    for rows, cin, cout in ((1, 1024, 512), (515, 771, 259), (512, 512, 512), (33003, 129, 257)):
        x, w, b = _rand(gpu, (rows, cin), dt, 1), _rand(gpu, (cin, cout), dt, 2, 0.05), _rand(gpu, (cout,), dt, 3)
        g = _rand(gpu, (rows, cout), dt, 4)

        def step():
            out, z = m.dense(x, w, b, activation="gelu", return_preact=True)
            return (out, z) + m.dense_grad(x, w, g, biases=b, activation="gelu", preact=z)

        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b_) for a, b_ in zip(other, want))
        graphs = []
        for _ in range(2):                             # two graphs of the same step, replayed in turn
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                outs = step()
            graphs.append((gr, outs))
        for turn in range(3):
            x.copy_(_rand(gpu, x.shape, dt, 10 + turn))
            eager = [t.clone() for t in step()]
            for gr, outs in graphs:
                gr.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b_) for a, b_ in zip(outs, eager))


@pytest.mark.gpu
def test_refused_arguments(gpu):
    m = _mod()
    x, w, g = torch.zeros(4, 6, device=gpu), torch.zeros(6, 8, device=gpu), torch.zeros(4, 8, device=gpu)
    for bad in (dict(inputs=x.double()), dict(inputs=x.int()), dict(weights=w.half()), dict(weights=w[:5]), dict(weights=w[None]),
                dict(biases=torch.zeros(7, device=gpu)), dict(biases=torch.zeros(8, device=gpu).half()), dict(biases=torch.zeros(8)),
                dict(residual=torch.zeros(4, 7, device=gpu)), dict(residual=g.half()), dict(activation="tanh"),
                dict(inputs=torch.zeros((), device=gpu)), dict(residual=torch.zeros(1, 8, device=gpu))):
        with pytest.raises(ValueError):
            m.dense(**{**dict(inputs=x, weights=w), **bad})
    for bad in (dict(grad_out=g[:3]), dict(grad_out=g.half()), dict(activation="relu"), dict(activation="relu", preact=g[:, :7]),
                dict(activation="relu", preact=g.cpu()), dict(needs=(True,))):
        with pytest.raises(ValueError):
            m.dense_grad(**{**dict(inputs=x, weights=w, grad_out=g), **bad})


# ------------------------------------------------------------------------------------------------ GPU: as they are used
@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_a_training_step_of_a_residual_block(gpu, dt):
    """Two layers with a residual around them, their gradients, and the clipping of all of them, against 64-bit autograd on
    the CPU.  16-bit: every intermediate is rounded to the type, half a step each; with some six roundings between input and
    gradient of terms of one size, 16 half steps of the tensor's largest value cover them.  fp32: the sums' errors."""
    m, c = _mod(), pkg("utils.tf_ops.gradients.tf_gradients")
    rows, ch, wide = 96, 64, 200
    x, w1, b1 = _rand(gpu, (rows, ch), dt, 1), _rand(gpu, (ch, wide), dt, 2, ch ** -0.5), _rand(gpu, (wide,), dt, 3, 0.1)
    w2, b2, g = _rand(gpu, (wide, ch), dt, 4, wide ** -0.5), _rand(gpu, (ch,), dt, 5, 0.1), _rand(gpu, (rows, ch), dt, 6)
    h, z = m.dense(x, w1, b1, activation="silu", return_preact=True)
    y = m.dense(h, w2, b2, residual=x)
    dh, dw2, db2 = m.dense_grad(h, w2, g, biases=b2)
    dx, dw1, db1 = m.dense_grad(x, w1, dh, biases=b1, activation="silu", preact=z)
    clipped, norm = c.clip_by_global_norm([dw1, db1, dw2, db2], 5.0)
    t = [v.double().cpu().requires_grad_() for v in (x, w1, b1, w2, b2)]
    yr = torch.nn.functional.silu(t[0] @ t[1] + t[2]) @ t[3] + t[4] + t[0]
    grads = torch.autograd.grad(yr, t, g.double().cpu())
    tol = 16 * _half(dt) if dt != torch.float32 else 2 * _sum_bound(wide) * 16

    def close(got, want, what):
        assert float((got.double().cpu() - want).abs().max()) <= tol * float(want.abs().max()), what

    close(y, yr.detach(), "y")
    close(dx + g, grads[0], "dx")                      # the residual's share is grad_out itself
    ref = math.sqrt(sum(float(v.pow(2).sum()) for v in grads[1:]))
    assert abs(float(norm) - ref) <= tol * ref and ref > 5.0
    for got, want, what in zip(clipped, grads[1:], ("w1", "b1", "w2", "b2")):
        close(got, want * (5.0 / ref), what)


def _held(d, dt):
    """How far the two planes of a 16-bit dz may be from it.  bf16: truncated to 8 bits, a step of 2^-7 of its power of two is left, of
    which 8 bits are rounded: 2^-16.  fp16: 11 and 11 bits, 2^-22, and the second plane's smallest number over 2048, 2^-35."""
    return {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}[dt] * d.abs() + 2.0 ** -35 * (dt == torch.float16)


def _check_unrounded(x, w, g, act, z, dx, dw, db):
    """As _check_grad, with a dz that is not rounded to the type."""
    gd = g.double()
    d = gd * _slope64(z.double(), act)
    dd = 0 * d if act is None else 32 * U * gd.abs() * (1 + z.double().abs()) + _tiny(torch.float32)
    dr = dd if act in (None, "relu") else dd + _held(d, x.dtype)
    wt, xt = w.double().t().contiguous(), x.double().t().contiguous()
    for got, want, bound, what in (
            (dx, lambda: d @ wt, lambda: (_sum_bound(w.shape[1]) * (d.abs() + dr) + dr) @ wt.abs(), "grad_inputs"),
            (dw, lambda: xt @ d, lambda: xt.abs() @ (_sum_bound(x.shape[0]) * (d.abs() + dr) + dr), "grad_weights"),
            (db, lambda: d.sum(0), lambda: (_sum_bound(x.shape[0]) * (d.abs() + dd) + dd).sum(0), "grad_biases")):
        if got is not None:
            want, bound = want(), bound()
            _within(got, want, _half(got.dtype) * (want.abs() + bound) + bound + _tiny(got.dtype), what)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_slopes_are_not_rounded(gpu, dt, size):
    """What is left are the fp32 sums and one rounding per result."""
    m = _mod()
    rows, cin, cout = size
    i = SIZES.index(size)
    for act in (ACTS[2 + i % 3], ACTS[i % 2]):
        x, w = _rand(gpu, (rows, cin), dt, i), _rand(gpu, (cin, cout), dt, 10 + i, math.sqrt(2.0 / cin))
        g, z = _rand(gpu, (rows, cout), dt, 20 + i, 0.05), _rand(gpu, (rows, cout), dt, 30 + i)
        b = torch.empty(cout, dtype=(dt, torch.float32)[i % 2], device=gpu)
        dx, dw, db = m.dense_grad(x, w, g, biases=b, activation=act, preact=z)
        assert dx.dtype == dw.dtype == dt and db.dtype == b.dtype
        _check_unrounded(x, w, g, act, z, dx, dw, db)
        only = m.dense_grad(x, w, g, activation=act, preact=z, needs=(False, True))
        assert only[0] is None and torch.equal(only[1], dw) and only[2] is None
        only = m.dense_grad(x, w, g, activation=act, preact=z, needs=(True, False))
        assert only[1] is None and torch.equal(only[0], dx) and only[2] is None


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_slopes_rounded_where_the_caller_says_so(gpu, dt, size):
    m = _mod()
    rows, cin, cout = size
    i = SIZES.index(size)
    act = ACTS[(i + 3) % 5]
    x, w = _rand(gpu, (rows, cin), dt, i), _rand(gpu, (cin, cout), dt, 10 + i, math.sqrt(2.0 / cin))
    g, z = _rand(gpu, (rows, cout), dt, 20 + i, 0.05), _rand(gpu, (rows, cout), dt, 30 + i)
    b = torch.empty(cout, dtype=(dt, torch.float32)[i % 2], device=gpu)
    dx, dw, db = m.dense_grad(x, w, g, biases=b, activation=act, preact=z, round_slopes=True)
    _check_grad(x, w, g, act, z, dx, dw, db)
    for needs in ((True, False), (False, True)):
        only = m.dense_grad(x, w, g, activation=act, preact=z, needs=needs, round_slopes=True)
        assert all(a is None or torch.equal(a, b_) for a, b_ in zip(only, (dx, dw, db)))
    if dt == torch.float32 or act in (None, "relu"):   # nothing is rounded there either way
        for a, b_ in zip((dx, dw, db), m.dense_grad(x, w, g, biases=b, activation=act, preact=z)):
            assert torch.equal(a, b_)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [(3, 64, 40), (300, 100, 260), (4, 64, 1100), (600, 500, 400), (1100, 1100, 1100), (1200, 1104, 1112)])
def test_small_slopes_and_infinite_factors(gpu, size, dt):
    """Gradients near the end of fp16's range keep their bits in the sums over many rows.  Infinite inputs, weights and gradients give
    the infinities of the product's sign and NaN where an infinity meets 0 or its opposite."""
    m = _mod()
    rows, cin, cout = size
    inf = float("inf")
    for act in ACTS[2:]:
        x, w = _rand(gpu, (rows, cin), dt, 1), _rand(gpu, (cin, cout), dt, 2)
        g, z = _rand(gpu, (rows, cout), dt, 3, 2e-6), _rand(gpu, (rows, cout), dt, 4, 2.0)
        b = torch.empty(cout, dtype=torch.float32, device=gpu)
        _check_unrounded(x, w, g, act, z, *m.dense_grad(x, w, g, biases=b, activation=act, preact=z))
        # now dz of a size that the first plane has, and no exact one
        g, z = _rand(gpu, (rows, cout), dt, 5), _rand(gpu, (rows, cout), dt, 6).clamp(-0.6, 0.6)
        g = torch.where(g.abs() < 1e-2, torch.ones((), dtype=dt, device=gpu), g)
        z[0, :3], g[0, :3] = 0.0, 1.0                  # and some exact ones: slope 1 / 2
        w[5, 7], w[7, 7], x[1, 3], x[rows - 1, 5] = inf, -inf, inf, -inf
        w[9, 2] = 0.0
        g[2, 4], g[2, 2] = inf, -inf
        dx, dw, db = m.dense_grad(x, w, g, biases=b, activation=act, preact=z)
        d = g.double() * _slope64(z.double(), act)
        big = torch.finfo(dt).max
        for got, want in ((dx, d @ w.double().t().contiguous()), (dw, x.double().t().contiguous() @ d), (db, d.sum(0))):
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            for s in (1, -1):
                assert torch.equal(got == s * inf, want == s * inf)
            assert float(want[torch.isfinite(want)].abs().max()) < big / 2


@pytest.mark.gpu
def test_more_work_items_than_a_grid_has(gpu):
    """Grids end at 2^32 work items: narrow layers of very many rows, and weight gradients of very many elements, have more.
    What lies behind the first launch's share is looked at, and the first rows."""
    m = _mod()
    dt = torch.bfloat16

    def ends(t, rows):
        return torch.cat([t[:100], t[rows // 2 - 50:rows // 2 + 50], t[-100:]])

    # forward: blocks of 32 rows by sixteen waves
    rows, cin = (1 << 27) + 70, 136
    x, w = torch.zeros(rows, cin, dtype=dt, device=gpu), _rand(gpu, (cin, 3), dt, 1)
    for i, at in enumerate((0, rows // 2 - 50, rows - 100)):
        x[at:at + 100] = _rand(gpu, (100, cin), dt, 10 + i)
    out = m.dense(x, w)
    _check_forward(ends(x, rows), w, None, None, None, ends(out, rows), None)
    assert not bool(out[100:rows // 2 - 50].any()) and not bool(out[rows // 2 + 50:-100].any())
    del x, out
    torch.cuda.empty_cache()
    # grad_inputs: blocks of 32 rows by eight waves, grad_weights in front or behind
    rows, cout = (1 << 28) + 70, 72
    x, w = torch.zeros(rows, 3, dtype=dt, device=gpu), _rand(gpu, (3, cout), dt, 2)
    g = torch.zeros(rows, cout, dtype=dt, device=gpu)
    for i, at in enumerate((0, rows // 2 - 50, rows - 100)):
        g[at:at + 100], x[at:at + 100] = _rand(gpu, (100, cout), dt, 20 + i), _rand(gpu, (100, 3), dt, 30 + i)
    dx, dw, db = m.dense_grad(x, w, g, biases=torch.empty(cout, device=gpu))
    _check_grad(ends(x, rows), w, ends(g, rows), None, None, ends(dx, rows), dw, db)
    assert not bool(dx[100:rows // 2 - 50].any()) and not bool(dx[rows // 2 + 50:-100].any())
    only = m.dense_grad(x, w, g, needs=(True, False))[0]
    assert torch.equal(only, dx)
    del x, g, dx, only
    torch.cuda.empty_cache()
    # grad_weights: 2^34 elements and more
    rows, cin, cout = 72, (1 << 17) + 40, 1 << 17
    x, g = _rand(gpu, (rows, cin), torch.float32, 3), _rand(gpu, (rows, cout), torch.float32, 4)
    _, dw, _ = m.dense_grad(x, torch.empty(cin, cout, device=gpu), g, needs=(False, True))
    for at in (0, cin // 2 - 20, cin - 40):
        _check_grad(x[:, at:at + 40].contiguous(), g, g, None, None, None, dw[at:at + 40], None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("size", [(3, 64, 40), (300, 100, 260), (600, 500, 400), (1100, 1100, 1100), (1200, 1104, 1112)])
def test_slopes_at_infinite_preactivations(gpu, size, act, dt):
    """The slope is 0 at -infinity and 1 at +infinity, in every kernel that forms one.  (The oracle takes z = -+60 there, where
    the slopes are 0 and 1 to more than 64 bits' worth of fp32.)"""
    m = _mod()
    rows, cin, cout = size
    x, w = _rand(gpu, (rows, cin), dt, 1), _rand(gpu, (cin, cout), dt, 2, cin ** -0.5)
    g, z = _rand(gpu, (rows, cout), dt, 3), _rand(gpu, (rows, cout), dt, 4)
    inf = float("inf")
    z[0, ::3], z[0, 1::3], z[rows - 1, cout - 1], z[rows // 2, 0] = inf, -inf, -inf, inf
    finite = z.clamp(-60, 60)
    b = torch.empty(cout, dtype=torch.float32, device=gpu)
    _check_grad(x, w, g, act, finite, *m.dense_grad(x, w, g, biases=b, activation=act, preact=z))
    _check_grad(x, w, g, act, finite, None, None, m.dense_grad(x, w, g, biases=b, activation=act, preact=z, needs=(False, False))[2])
    z[1, 2] = float("nan")                             # a NaN still comes through, in its row and column
    dx, dw, db = m.dense_grad(x, w, g, biases=b, activation=act, preact=z)
    assert bool(torch.isnan(dx[1]).all()) and bool(torch.isnan(dw[:, 2]).all()) and bool(torch.isnan(db[2]))
    assert int(torch.isnan(dx).any(1).sum()) == 1 and int(torch.isnan(dw).any(0).sum()) == 1 and int(torch.isnan(db).sum()) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS[1:])
def test_a_preactivation_that_fp16_keeps_as_an_infinity(gpu, act):
    """z of +-10^5 is finite in the forward pass's fp32 and +-infinity in the fp16 that the backward pass gets."""
    m = _mod()
    dt = torch.float16
    x, w, g = torch.ones(4, 8, dtype=dt, device=gpu), _rand(gpu, (8, 16), dt, 1), _rand(gpu, (4, 16), dt, 2)
    w[:, 3], w[:, 5] = -12500.0, 2.0                   # -99968 (12500 is no fp16 number, 12496 is), 16
    x[2] = 1.0 / 8
    out, z = m.dense(x, w, activation=act, return_preact=True)
    assert float(z[0, 3]) == -float("inf") and float(z[2, 3]) == float(w[0, 3])
    assert bool((out[:, 3] == 0).all()) and bool(torch.isfinite(out).all())
    dx, dw, db = m.dense_grad(x, w, g, biases=torch.empty(16, device=gpu), activation=act, preact=z)
    _check_grad(x, w, g, act, z.clamp(-60, 60), dx, dw, db)
    assert bool((dw[:, 3] == 0).all()) and float(db[3]) == 0


def test_rows_of_no_columns_keep_their_number():
    m = _mod()
    for shape in ((2, 3, 0), (0,), (6, 0), (2, 0, 3, 0)):
        t, _, ld = m._rows(torch.zeros(shape), 0)
        assert t.shape == (math.prod(shape[:-1]), 0) and ld >= 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_no_input_channels_with_any_leading_dimensions(gpu, dt):
    m = _mod()
    w, b = torch.empty(0, 7, dtype=dt, device=gpu), _rand(gpu, (7,), dt, 1)
    for lead in ((), (3,), (2, 3), (2, 1, 5), (2, 0, 3)):
        x, r = torch.empty(lead + (0,), dtype=dt, device=gpu), _rand(gpu, lead + (7,), dt, 2)
        out, z = m.dense(x, w, b, activation="silu", residual=r, return_preact=True)
        assert out.shape == lead + (7,) and torch.equal(z, b.expand(lead + (7,)))
        want = _act64(b.double(), "silu") + r.double()
        _within(out, want, _half(dt) * want.abs() + 40 * U * (1 + want.abs() + r.double().abs()) + _tiny(dt), "out")
        assert not bool(m.dense(x, w).any())
        dx, dw, db = m.dense_grad(x, w, r, biases=b)
        assert dx.shape == x.shape and dw.shape == (0, 7)
        rd = r.double().view(-1, 7)
        _within(db, rd.sum(0), _half(dt) * rd.sum(0).abs() + 8 * U * rd.abs().sum(0) + _tiny(dt), "grad_biases")


def test_scratch_of_empty_layers():
    """Gradients that an empty layer does not have need no scratch, and asking for it is no error."""
    lib = pkg("utils._native").lib()
    n = ctypes.c_ulong()
    for dtype in range(3):
        for act in (0, 1, 4):
            for want in range(8):
                for rows, cin, cout in ((0, 5, 7), (3, 0, 7), (3, 5, 0), (0, 0, 7), (0, 5, 0), (3, 0, 0), (0, 0, 0), (4000, 0, 4000),
                                        (0, 4000, 4000), (4000, 4000, 0)):
                    n.value = 1
                    assert lib.sa_dense_backward_ws(dtype, rows, cin, cout, act, want, 7, ctypes.byref(n)) == 0
                    # the column sums of rows that are there are all that takes any
                    assert n.value == 0 or (want & 4 and rows and cout and not cin)


def test_the_c_entries_refuse_addresses_inside_an_element_and_unaligned_scratch():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses below: only where nothing could be launched on them")
    lib = pkg("utils._native").lib()
    n = ctypes.c_ulong()
    p = 1 << 20                                        # an address that is never dereferenced: every call below is refused
    for dtype, off in ((0, 1), (0, 2), (1, 1), (2, 1)):
        ok = dict(x=p, w=p, bias=p, res=p, y=p, pre=p)
        for name in ok:
            a = {**ok, name: p + off}
            assert lib.sa_dense_forward(dtype, 4, 8, 8, a["x"], 8, a["w"], 8, a["bias"], 0, a["res"], 8, 1, a["y"], a["pre"], None, 0,
                                        None) == -1, (dtype, off, name)
        ok = dict(x=p, w=p, g=p, z=p, dx=p, dw=p, db=p)
        for name in ok:
            a = {**ok, name: p + off}
            assert lib.sa_dense_backward(dtype, 4, 8, 8, a["x"], 8, a["w"], 8, a["g"], 8, a["z"], 8, 1, a["dx"], a["dw"], a["db"], 0,
                                         None, 0, None) == -1, (dtype, off, name)
    assert lib.sa_dense_forward(1, 4, 8, 8, p, 8, p, 8, p + 2, 1, None, 0, 0, p, None, None, 0, None) == -1      # fp32 bias, fp32 db
    assert lib.sa_dense_backward(1, 4, 8, 8, p, 8, p, 8, p, 8, None, 0, 0, p, p, p + 2, 1, None, 0, None) == -1
    assert lib.sa_dense_forward_ws(1, 400, 4096, 8, 3, ctypes.byref(n)) == 0 and n.value > 0
    for off in (2, 16, 128):
        assert lib.sa_dense_forward(1, 400, 4096, 8, p, 4096, p, 8, None, 0, None, 0, 0, p, None, p + off, n.value, None) == -1
    assert lib.sa_dense_backward_ws(1, 4000, 1000, 1000, 0, 7, 7, ctypes.byref(n)) == 0 and n.value > 0
    for off in (2, 16, 128):
        assert lib.sa_dense_backward(1, 4000, 1000, 1000, p, 1000, p, 1000, p, 1000, None, 0, 0, p, p, p, 0, p + off, n.value, None) == -1


# ------------------------------------------------------------------------------- large fp32 products: bits and ranges of a factor
def _planes(v):
    """v = h + m + l + what 27 bits do not hold, each plane bf16 (CPU)."""
    out = []
    for _ in range(3):
        p = v.to(torch.bfloat16).float()
        out.append(p)
        v = v - p
    return out


PLANE_PRODUCTS = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]
# Of |x w|.  Left out are m l and l m, at most 2^-27 each (m is within 2^-9 of the factor, l within 2^-18), and what is behind
# either factor's third plane, 2^-27 each: 2^-25 or U / 2.  An addition to a sum of the product's size is off by a step, 2 U, at
# the most, one below 2^-8 of that size by nothing that counts.  There are up to four of those: the split kernel's last block adds
# h h third, and m m, h m and h l behind it; elsewhere h h comes last.  8.5 U, against 2^-18 = 64 U and more of a whole l h or m m.
SINGLE_TERM = 9 * U


def _factors(shape, seed, device="cpu"):
    """Random 24-bit mantissas, signs, and exponents from -20 to 20; a few with planes as large as they get."""
    g = torch.Generator().manual_seed(seed)
    v = (1 + torch.rand(shape, generator=g, dtype=torch.float64)).float() * torch.exp2(torch.randint(-20, 21, shape, generator=g).float())
    v = torch.where(torch.rand(shape, generator=g) < 0.5, -v, v)
    v.view(-1)[::7] = 1 + 2.0 ** -8 * (1 - 2.0 ** -7) + 2.0 ** -17
    return v.to(device)


def test_a_missing_plane_product_shows_in_a_single_term():
    """The bound below sees each of the six products: without any one of them a CPU emulation is outside."""
    x, w = _factors((4000,), 1), _factors((4000,), 2)
    px, pw = _planes(x), _planes(w)
    want = x.double() * w.double()
    for missing in [None] + PLANE_PRODUCTS:
        got = sum(px[a].double() * pw[b].double() for a, b in PLANE_PRODUCTS if (a, b) != missing).float().double()
        inside = bool(((got - want).abs() <= SINGLE_TERM * want.abs()).all())
        assert inside == (missing is None), missing


SINGLE_FORWARD = {"split": (2048, 512, 8192), "tiles": (2048, 512, 2048)}
SINGLE_WEIGHTS = {"split": (300, 4096, 4096), "tiles": (300, 8192, 1024), "pieces": (4096, 1024, 1024)}


def test_both_kernels_of_large_fp32_products_are_met():
    """By their scratch: the tiles have planes of both factors there, the split kernel of the second only."""
    lib = pkg("utils._native").lib()
    n = ctypes.c_ulong()
    up = lambda v, m: (v + m - 1) // m * m  # noqa: E731
    planes = lambda rows, cols: up(6 * rows * up(cols, 64), 256)  # noqa: E731
    for kernel, (rows, cin, cout) in SINGLE_FORWARD.items():
        assert lib.sa_dense_forward_ws(0, rows, cin, cout, 3, ctypes.byref(n)) == 0
        assert n.value == planes(cin, cout) + (planes(rows, cin) if kernel == "tiles" else 0)
    for kernel, (rows, cin, cout) in SINGLE_WEIGHTS.items():
        assert lib.sa_dense_backward_ws(0, rows, cin, cout, 0, 2, 7, ctypes.byref(n)) == 0
        least = planes(rows, cout) + (planes(rows, cin) if kernel == "tiles" else 0)
        assert n.value > least if kernel == "pieces" else n.value == least


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", sorted(SINGLE_FORWARD))
def test_every_bit_of_a_single_term(gpu, kernel):
    """One nonzero factor per sum: no other term hides the bits of its product."""
    m = _mod()
    rows, cin, cout = SINGLE_FORWARD[kernel]
    x, w = torch.zeros(rows, cin, device=gpu), _factors((cin, cout), 1, gpu)
    at = torch.arange(rows, device=gpu) * 37 % cin
    v = _factors((rows,), 2, gpu)
    x[torch.arange(rows, device=gpu), at] = v
    want = v.double()[:, None] * w.double()[at]
    _within(m.dense(x, w), want, SINGLE_TERM * want.abs(), "out")


@pytest.mark.gpu
@pytest.mark.parametrize("size", sorted(SINGLE_WEIGHTS.values()))
def test_every_bit_of_a_single_term_of_the_gradient(gpu, size):
    m = _mod()
    rows, cin, cout = size
    r = torch.arange(rows, device=gpu)
    # grad_inputs: one nonzero grad_out per row
    g, w, x = torch.zeros(rows, cout, device=gpu), _factors((cin, cout), 1, gpu), _factors((rows, cin), 2, gpu)
    at, v = r * 37 % cout, _factors((rows,), 3, gpu)
    g[r, at] = v
    want = v.double()[:, None] * w.double().t().contiguous()[at]
    _within(m.dense_grad(x, w, g, needs=(True, False))[0], want, SINGLE_TERM * want.abs(), "grad_inputs")
    # grad_weights: one nonzero input per channel
    g, x = _factors((rows, cout), 4, gpu), torch.zeros(rows, cin, device=gpu)
    c = torch.arange(cin, device=gpu)
    at, v = (c * 41 + 5) % rows, _factors((cin,), 5, gpu)
    x[at, c] = v
    want = v.double()[:, None] * g.double()[at]
    for needs in ((False, True), (True, True)):
        _within(m.dense_grad(x, w, g, needs=needs)[1], want, SINGLE_TERM * want.abs(), "grad_weights")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_negative_tails_are_relatively_right(gpu, act):
    """fp32, one channel of weight 1, so z is the input.  The value in the tail is an exponential: a rounding of its exponent by u
    relative shows times the exponent.  GELU: exponent z^2 / 2, two roundings and a constant: 1.5 z^2 u; polynomial, reciprocals
    (two steps each), exponential and products: 24 u.  SiLU: 2 |z| u and 12 u.  Tanh form: exponent 2 sqrt(2/pi) (z + 0.044715 z^3)
    with seven roundings and two constants: 10 u of it, and 12 u.  The slopes are sums of two such terms,
    the second with s (1 - s): twice the error of s."""
    m = _mod()
    low = {"gelu": -12.8, "gelu_tanh": -9.8, "silu": -85.0}[act]
    x = torch.linspace(low, 0, 20001, device=gpu)[:, None]
    one = torch.ones(1, 1, device=gpu)
    z = x.double()
    e = {"gelu": 24 + 1.5 * z * z, "silu": 12 + 2 * z.abs(), "gelu_tanh": 12 + 10 * 1.5957691216 * (z.abs() + 0.044715 * z.abs() ** 3)}[act] * U
    # (tanh and ndtr of torch lose the tails: the formulas without a difference)
    if act == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        second = z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        u, du = (z, 1.0) if act == "silu" else (2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3),
                                                2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z))
        p = torch.exp(u) / (1 + torch.exp(u))
        second = z * p / (1 + torch.exp(u)) * du
    out, pre = m.dense(x, one, activation=act, return_preact=True)
    assert torch.equal(pre, x)
    _within(out, z * p, e * (z * p).abs() + 1e-45, "out")
    slope = m.dense_grad(x, one, torch.ones_like(x), activation=act, preact=x, needs=(True, False))[0]
    _within(slope, p + second, (2 * e + 8 * U) * (p + second.abs()), "slope")


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(70, 129, 65), (2048, 512, 2048), (2048, 512, 8192)])
def test_tiny_fp32_factors(gpu, size):
    """Large products hold a fp32 factor to 2^-24 of itself or to 2^-134, half of the smallest step of its planes, whichever is
    larger; small ones to all of its bits.  And an infinity times anything but 0 and NaN is an infinity.
    (A factor below 2^-126 enters the matrix instructions unnormalised, as 2^-126 times a fraction: a sum with it keeps 24 bits from
    2^-126 times the other factor down, so that each of the six products may be off by 2^-149 times the other factor.)"""
    m = _mod()
    held = 2.0 ** -134 + 6 * 2.0 ** -149
    rows, cin, cout = size
    r = torch.arange(rows, device=gpu)
    at = r * 37 % cin
    w = _factors((cin, cout), 1, gpu) * 2.0 ** 70      # 2^50 to 2^91
    for e in (-100, -108, -114, -120, -126):
        v = _factors((rows,), 2, gpu).sign() * (1 + torch.rand(rows, generator=torch.Generator().manual_seed(3))).to(gpu) * 2.0 ** e
        x = torch.zeros(rows, cin, device=gpu)
        x[r, at] = v
        want = v.double()[:, None] * w.double()[at]
        step = held * w.double().abs()[at] * (rows > 100)
        _within(m.dense(x, w), want, SINGLE_TERM * want.abs() + step, "out")
        # the same with the factors' parts exchanged: W tiny, X large
        tiny = torch.ldexp(_factors((cin, cout), 4, gpu), torch.tensor(e - 20, device=gpu))
        x[r, at] = _factors((rows,), 5, gpu) * 2.0 ** 100
        want = x[r, at].double()[:, None] * tiny.double()[at]
        step = held * x[r, at].double().abs()[:, None] * (rows > 100)
        _within(m.dense(x, tiny), want, SINGLE_TERM * want.abs() + step, "out, tiny weights")
    # infinities
    inf = float("inf")
    tiny = torch.tensor([1e-30, 2.0 ** -126, 2.0 ** -133, 2.0 ** -134, 1.5 * 2.0 ** -134, 2.0 ** -135, 2.0 ** -149, 0.0, 1e-40], dtype=torch.float64)
    tiny = torch.cat([tiny, -tiny]).float().to(gpu)
    assert int((tiny != 0).sum()) == 16
    ones = torch.ones(rows, device=gpu)
    ones[1::2] = -1

    def signs(got, want, what):
        for a, b in ((torch.isnan(got), torch.isnan(want)), (got == inf, want == inf), (got == -inf, want == -inf)):
            assert torch.equal(a, b), what

    x, w = torch.zeros(rows, cin, device=gpu), tiny.repeat(cin * cout // 18 + 1)[:cin * cout].view(cin, cout).contiguous()
    x[r, at] = ones * inf
    signs(m.dense(x, w), (ones * inf)[:, None] * w[at], "infinite inputs, tiny weights")
    g = torch.zeros(rows, cout, device=gpu)
    to = r * 37 % cout
    g[r, to] = ones * inf
    signs(m.dense_grad(x, w, g, needs=(True, False))[0], (ones * inf)[:, None] * w.t()[to], "infinite grad_out, tiny weights")
    x[r, at] = tiny.repeat(rows // 18 + 1)[:rows]
    full = torch.where(x == 0, 2.0 ** -140, x)         # tiny factors all along a row, of one sign
    full = full.abs() * ones[:, None]
    w = torch.full((cin, cout), inf, device=gpu)
    w[:, 1::2] = -inf
    signs(m.dense(full, w), (ones * inf)[:, None] * w[:1], "tiny inputs, infinite weights")
    c = torch.arange(cin, device=gpu)
    x, g = torch.zeros(rows, cin, device=gpu), torch.full((rows, cout), 2.0 ** -141, device=gpu)
    x[(c * 41 + 5) % rows, c] = inf
    signs(m.dense_grad(x, w, g, needs=(False, True))[1], torch.full((cin, cout), inf, device=gpu), "infinite inputs, tiny grad_out")


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(70, 129, 65), (2048, 512, 2048), (2048, 512, 8192)])
def test_fp32_products_near_the_largest_number(gpu, size):
    # the first planes may be larger than their factors, by 2^-8 each: a product up to the largest number / 1.008 does not overflow
    m = _mod()
    rows, cin, cout = size
    g = torch.Generator(device=gpu).manual_seed(1)
    r = torch.arange(rows, device=gpu)
    at = r * 37 % cin
    x, w = torch.zeros(rows, cin, device=gpu), 1 - 0.1 * torch.rand(cin, cout, generator=g, device=gpu)
    x[r, at] = (torch.finfo(torch.float32).max / 1.008) * (1 - 0.1 * torch.rand(rows, generator=g, device=gpu))
    want = x[r, at].double()[:, None] * w.double()[at]
    _within(m.dense(x, w), want, SINGLE_TERM * want.abs(), "out")
