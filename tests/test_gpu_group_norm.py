"""Group norm with activation and dropout (ba_norm_forward / _backward)
against its definition in 64 bits.

Tolerances, with u = 2^-24 (half an fp32 step, relative), R the largest
|x - mean| of a group and M its largest |x|:
* statistics: a thread sums at most 64 values about its own first one, and
  trees of at most 8 levels and double sums follow, so the mean is within
  (64 + 8) u 2R + 2 u M and the variance within 2 (64 + 8) u of itself; taken
  together as 160 u: z is within K = rstd |w| (160 u R + 4 u M) + 160 u |z|;
* the activations' slopes are at most 1.13 (and their second derivatives at
  most 1), the hardware's exp and reciprocal and the erf are within 16 u of
  their value plus 16 u absolute: y within 1.13 K + 16 u (|y| + |z| + 1),
  times dropout's scale;
* dz within |dy| (K + 16 u (1 + |z|)) scale;
* a channel's sums (fp32 in runs of at most 64 and trees, then double): the
  errors of their terms, plus 80 u of the sum of magnitudes;
* dx: the errors of dz and of the two group means, each times rstd |w|, plus
  16 u of the terms.
Each result is then rounded once to its type: eps / 2 of its value.
The rectifiers' slopes jump at z = 0, so where |z| is within K of it the
incoming gradient is zero in these tests."""
from __future__ import annotations

import pytest
import torch

import feature_ref as R

pytestmark = pytest.mark.gpu

U = 2.0**-24


def _x(shape, dtype, layout, seed=0, offset=0.5, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    B, C = shape[:2]
    x = torch.randn(*shape, generator=g) * spread + offset * torch.randn(1, C, 1, 1, 1, generator=g)
    x = x.to(dtype).cuda()
    return x.contiguous(memory_format=torch.channels_last_3d) if layout == "last" else x


def _params(C, kind, seed=5):
    g = torch.Generator().manual_seed(seed)
    w, b = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    if kind is None:
        return None, None
    return w.to(kind).cuda(), b.to(kind).cuda()


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _bounds(x, groups, w, eps, z):
    """K of the module's notes, and rstd |w|, for every value."""
    B, C = x.shape[:2]
    r = x.reshape(B, groups, -1)
    m = r.mean(-1, keepdim=True)
    big = (r - m).abs().amax(-1, keepdim=True).expand_as(r).reshape(x.shape)
    top = r.abs().amax(-1, keepdim=True).expand_as(r).reshape(x.shape)
    rstd = (1 / torch.sqrt(((r - m) ** 2).mean(-1, keepdim=True) + eps)).expand_as(r).reshape(x.shape)
    aw = rstd if w is None else rstd * w.abs().reshape(1, C, 1, 1, 1)
    return aw * (160 * U * big + 4 * U * top) + 160 * U * z.abs(), aw


def _gmean(t, groups):
    B = t.shape[0]
    return t.reshape(B, groups, -1).mean(-1, keepdim=True).expand(B, groups, t[0].numel() // groups) \
        .reshape(t.shape)


def _run(ba, shape, dtype, layout, groups, act, kind=torch.float32, p=0.0, seed=3, eps=1e-5,
         offset=0.5, spread=1.0, x=None, slope=0.01):
    C = shape[1]
    x = _x(shape, dtype, layout, offset=offset, spread=spread) if x is None else x
    w, b = _params(C, kind)
    leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_()
              for t in (x, w, b) if t is not None]
    y = ba.ops.group_norm(leaves[0], groups, *(leaves[1:] or (None, None)), eps=eps,
                          activation=act, negative_slope=slope, p=p, seed=seed)
    assert y.dtype == dtype and y.shape == x.shape and y.stride() == x.stride()

    # the definition, on the CPU in 64 bits
    l64 = [t.detach().double().cpu().contiguous().requires_grad_() for t in leaves]
    f = R.factor(shape, p, seed) if p else None
    ref, z = R.norm(l64[0], groups, *(l64[1:] or (None, None)), eps=eps, act=act, slope=slope, f=f)
    z = z.detach()
    K, aw = _bounds(l64[0].detach(), groups, l64[1].detach() if w is not None else None, eps, z)
    scale = 1.0 if f is None else float(f.max())
    got = y.detach().double().cpu()
    if f is not None:
        assert torch.equal(got[f == 0], torch.zeros_like(got[f == 0]))
    tol = scale * (1.13 * K + 16 * U * (ref.detach().abs() + z.abs() + 1)) \
        + _half_step(dtype) * ref.detach().abs()
    assert ((got - ref.detach()).abs() <= tol).all(), \
        float(((got - ref.detach()).abs() / tol).max())

    # gradients
    g = torch.Generator().manual_seed(11)
    dy = torch.randn(*shape, generator=g).to(dtype)
    if act in ("relu", "leaky_relu"):
        dy = torch.where(z.abs() <= 2 * K, torch.zeros_like(dy), dy)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    refs = torch.autograd.grad(ref, l64, dy.double())
    zz = z.clone().requires_grad_()
    (slope_z,) = torch.autograd.grad(R.activation(zz, act, slope).sum(), zz)
    dout = dy.double() * (1.0 if f is None else f)
    dz = dout * slope_z
    e_dz = dout.abs() * (K + 16 * U * (1 + z.abs()))
    xh = R.norm(l64[0].detach(), groups, eps=eps)[0]
    e_xh = K / (1.0 if w is None else l64[1].detach().abs().reshape(1, C, 1, 1, 1)) \
        if w is None or bool((l64[1] != 0).all()) else K
    wv = torch.ones(1, C, 1, 1, 1, dtype=torch.float64) if w is None \
        else l64[1].detach().reshape(1, C, 1, 1, 1)
    t1, t2 = (wv * dz).abs(), (wv * dz * xh).abs()
    e1 = wv.abs() * e_dz + 80 * U * t1
    e2 = wv.abs() * (e_dz * xh.abs() + dz.abs() * e_xh) + 80 * U * t2
    rstd = aw / wv.abs() if w is not None else aw
    a2 = _gmean(t2, groups)
    tol_dx = rstd * (wv.abs() * e_dz + _gmean(e1, groups) + xh.abs() * _gmean(e2, groups)
                     + e_xh * a2 + 16 * U * (t1 + _gmean(t1, groups) + xh.abs() * a2)
                     + 160 * U * (t1 + _gmean(t1, groups) + xh.abs() * a2))
    _close(grads[0], refs[0], tol_dx + _half_step(dtype) * refs[0].abs())
    assert grads[0].stride() == x.stride()
    if w is not None:
        axes = (0, 2, 3, 4)
        e_w = e_dz * xh.abs() + dz.abs() * e_xh + 80 * U * (dz * xh).abs()
        _close(grads[1], refs[1], e_w.sum(axes) + _half_step(kind) * refs[1].abs())
        _close(grads[2], refs[2], (e_dz + 80 * U * dz.abs()).sum(axes)
               + _half_step(kind) * refs[2].abs())
    return y, grads


def _close(got, ref, tol):
    err = (got.double().cpu() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-300)).max())


SHAPES = [  # (shape, groups)
    ((1, 1, 1, 1, 1), 1), ((2, 4, 1, 1, 1), 2), ((2, 8, 1, 1, 3), 8), ((1, 8, 2, 2, 2), 1),
    ((2, 16, 3, 5, 7), 4), ((1, 4, 8, 8, 9), 2), ((2, 12, 5, 4, 4), 3), ((3, 33, 3, 3, 3), 11),
    ((1, 2, 9, 16, 32), 2), ((1, 5, 17, 19, 23), 1), ((1, 2056, 1, 2, 5), 8), ((2, 520, 2, 3, 3), 65),
    ((1, 1, 20, 20, 20), 1), ((2, 20, 1, 3, 43), 5), ((1, 64, 24, 20, 16), 8), ((1, 3, 31, 33, 35), 3),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("shape, groups", SHAPES)
def test_shapes(ba, shape, groups, layout, dtype):
    _run(ba, shape, dtype, layout, groups, "silu", eps=1e-2)


@pytest.mark.parametrize("act", [None, "relu", "leaky_relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_activations(ba, act, dtype, layout, p):
    for shape, groups in (((2, 16, 6, 7, 8), 4), ((2, 6, 5, 5, 5), 3)):
        _run(ba, shape, dtype, layout, groups, act, p=p, seed=2**40 + 1, slope=0.2)


@pytest.mark.parametrize("kind", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["first", "last"])
def test_params(ba, kind, layout):
    _run(ba, (2, 24, 4, 5, 6), torch.bfloat16, layout, 6, "gelu", kind=kind, p=0.1)
    x = _x((2, 24, 4, 5, 6), torch.float32, layout)
    w, b = _params(24, torch.float32)
    ops = ba.ops
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    assert torch.equal(ops.group_norm(x, 6, w), ops.group_norm(x, 6, w, zero))
    assert torch.equal(ops.group_norm(x, 6, None, b), ops.group_norm(x, 6, one, b))
    # a gradient for the weight alone, for x alone
    w.requires_grad_()
    (dw,) = torch.autograd.grad(ops.group_norm(x, 6, w, b).sum(), w)
    xr = x.clone(memory_format=torch.preserve_format).requires_grad_()
    full = torch.autograd.grad(ops.group_norm(xr, 6, w, b).sum(), [xr, w])
    assert torch.equal(dw, full[1])
    (dx,) = torch.autograd.grad(ops.group_norm(xr, 6, w.detach(), b).sum(), xr)
    assert torch.equal(dx, full[0])


@pytest.mark.parametrize("layout", ["first", "last"])
def test_offset_far_larger_than_spread(ba, layout):
    """Intensities of 1000 +- 0.1, with a corner far off them."""
    shape = (2, 8, 12, 13, 14)
    x = _x(shape, torch.float32, layout, offset=0.0, spread=0.1) + 1000.0
    _run(ba, shape, torch.float32, layout, 2, None, x=x)
    x[:, :, 0, 0, 0] = 0.0
    _run(ba, shape, torch.float32, layout, 2, None, x=x)


@pytest.mark.parametrize("layout", ["first", "last"])
def test_constant_groups(ba, layout):
    """A group without spread: xhat is zero, and the gradient finite."""
    shape = (2, 8, 5, 5, 5)
    x = torch.full(shape, 3.25, device="cuda")
    x = x.contiguous(memory_format=torch.channels_last_3d) if layout == "last" else x
    w, b = _params(8, torch.float32)
    x.requires_grad_()
    y = ba.ops.group_norm(x, 4, w, b, activation="silu")
    ref = R.activation(b.double().cpu(), "silu").reshape(1, 8, 1, 1, 1).expand(shape)
    assert ((y.detach().double().cpu() - ref).abs() <= 16 * U * (ref.abs() + 1)).all()
    (dx,) = torch.autograd.grad(y.sum(), x)
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("layout", ["first", "last"])
def test_nan_stays_in_its_group(ba, layout):
    shape = (2, 8, 5, 6, 7)
    x = _x(shape, torch.float32, layout)
    clean = ba.ops.group_norm(x, 4, activation="gelu")
    for bad in (float("nan"), float("inf")):
        v = x.clone(memory_format=torch.preserve_format)
        v[1, 5, 2, 3, 4] = bad
        y = ba.ops.group_norm(v, 4, activation="gelu")
        assert torch.isnan(y[1, 4:6]).all()
        keep = torch.ones(2, 8, dtype=torch.bool)
        keep[1, 4:6] = False
        assert torch.equal(y[keep.cuda()], clean[keep.cuda()])


def test_same_bits_every_time(ba):
    shape = (2, 32, 20, 21, 22)
    for layout in ("first", "last"):
        first = _run_bits(ba, shape, layout)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, _run_bits(ba, shape, layout)))


def _run_bits(ba, shape, layout):
    x = _x(shape, torch.bfloat16, layout).requires_grad_()
    w, b = _params(shape[1], torch.float32)
    w.requires_grad_(), b.requires_grad_()
    y = ba.ops.group_norm(x, 8, w, b, activation="silu", p=0.1, seed=4)
    return [y.detach()] + list(torch.autograd.grad(y, [x, w, b], _x(shape, torch.bfloat16, layout, 9)))


def test_gradients_against_differences(ba):
    """Central differences of the operator itself, in fp32 with a step of
    1/16: the third derivatives leave h^2 / 6 of a curvature of order one,
    rounding 2 |y|_1 u 2^4 / 2h."""
    shape = (1, 4, 3, 3, 3)
    x = _x(shape, torch.float32, "last").requires_grad_()
    w, b = _params(4, torch.float32)
    w.requires_grad_(), b.requires_grad_()
    c = _x(shape, torch.float32, "first", seed=2)

    def f(x_, w_, b_):
        y = ba.ops.group_norm(x_, 2, w_, b_, eps=0.1, activation="silu", p=0.2, seed=6)
        return (y.double() * c.double()).sum()

    grads = torch.autograd.grad(f(x, w, b), [x, w, b])
    h = 1 / 16
    for i, leaf in enumerate((x, w, b)):
        for j in range(0, leaf.numel(), 7 if i == 0 else 1):
            def at(step):
                args = [t.detach().clone(memory_format=torch.preserve_format) for t in (x, w, b)]
                flat = args[i].permute(0, 2, 3, 4, 1).reshape(-1) if i == 0 else args[i]
                flat[j] += step
                return float(f(*args))
            got = float((grads[i].permute(0, 2, 3, 4, 1).reshape(-1) if i == 0 else grads[i])[j])
            diff = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
            # fourth-order differences: h^4 / 30 of a fifth derivative, at most ~2e3 here
            assert abs(got - diff) <= 2e3 * h**4 / 30 + 1e-3


def test_empty_and_single(ba):
    w, b = _params(4, torch.float32)
    for shape in ((0, 4, 2, 2, 2), (2, 4, 0, 2, 2)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        ws, bs = w.clone().requires_grad_(), b.clone().requires_grad_()
        y = ba.ops.group_norm(x, 2, ws, bs, activation="silu", p=0.5, seed=1)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and not ws.grad.any() and not bs.grad.any()
    # one value a group: xhat is zero
    x = _x((2, 4, 1, 1, 1), torch.float32, "first").requires_grad_()
    y = ba.ops.group_norm(x, 4, w, b)
    assert torch.equal(y.detach(), b.reshape(1, 4, 1, 1, 1).expand(2, 4, 1, 1, 1))
    (dx,) = torch.autograd.grad(y.sum(), x)
    assert not dx.any()


def test_views_and_broadcast_gradients(ba):
    v = _x((2, 16, 6, 6, 6), torch.float32, "first")[:, 2:10, 1::2]
    y = ba.ops.group_norm(v, 4, activation="silu")
    assert torch.equal(y, ba.ops.group_norm(v.contiguous(), 4, activation="silu"))
    base = torch.randn(1 + 2 * 8 * 125, device="cuda").to(torch.bfloat16)
    u = base[1:].view(2, 8, 5, 5, 5)
    assert torch.equal(ba.ops.group_norm(u, 2), ba.ops.group_norm(u.clone(), 2))
    x = _x((2, 8, 4, 4, 4), torch.float32, "last").requires_grad_()
    one = torch.autograd.grad(ba.ops.group_norm(x, 2, activation="silu").sum(), x)[0]
    full = torch.autograd.grad(ba.ops.group_norm(x, 2, activation="silu"), x,
                               torch.ones(2, 8, 4, 4, 4, device="cuda"))[0]
    assert torch.equal(one, full)


def test_streams(ba):
    """Two streams at once, each with its own scratch."""
    xs = [_x((2, 32, 16, 16, 16), torch.bfloat16, "last", seed=i) for i in range(2)]
    want = [ba.ops.group_norm(x, 8, activation="silu") for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ba.ops.group_norm(xs[i], 8, activation="silu"))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_training_step_in_a_graph(ba):
    """Forward and backward captured once, replayed on other data and seeds;
    a second graph of the same operator is replayed in between."""
    shape = (2, 16, 8, 9, 10)
    static = _x(shape, torch.float32, "last").requires_grad_()
    w, b = (t.requires_grad_() for t in _params(16, torch.float32))
    seed = torch.tensor([7], dtype=torch.int64, device="cuda")
    dy = _x(shape, torch.float32, "last", seed=1)

    def step():
        # detached, so that no eager or captured graph of the leaves outlives its step
        y = ba.ops.group_norm(static, 4, w, b, activation="silu", p=0.2, seed=seed)
        return [y.detach()] + list(torch.autograd.grad(y, [static, w, b], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        with torch.no_grad():
            static.copy_(_x(shape, torch.float32, "last", seed=20 + k))
        seed.fill_(50 + k)
        for g, _ in graphs:
            g.replay()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_refusals(ba):
    x = torch.zeros(2, 6, 4, 4, 4, device="cuda")
    gn = ba.ops.group_norm
    for bad in (0, 4, -1):
        with pytest.raises(ValueError, match="groups"):
            gn(x, bad)
    with pytest.raises(ValueError, match="activation"):
        gn(x, 2, activation="tanh")
    with pytest.raises(ValueError, match="weight"):
        gn(x, 2, torch.ones(5, device="cuda"))
    with pytest.raises(ValueError, match="weight is on"):
        gn(x, 2, torch.ones(6))
    with pytest.raises(ValueError, match="bias"):
        gn(x, 2, torch.ones(6, device="cuda"), torch.ones(6, device="cuda").bfloat16())
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        gn(x, 2, torch.ones(6, device="cuda").half())
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        gn(x.double(), 2)
    with pytest.raises(ValueError, match="seed"):
        gn(x, 2, p=0.5)
    with pytest.raises(ValueError, match="eps"):
        gn(x, 2, eps=-1.0)
    with pytest.raises(ValueError, match="B,C,H,W,D"):
        gn(x[0], 2)
    y = gn(x.requires_grad_(), 2)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("shape, groups", [((1, 300, 1, 2, 5), 1), ((1, 8, 40, 40, 40), 1),
                                           ((2, 64, 24, 24, 24), 8), ((1, 2, 96, 64, 64), 2)])
def test_statistics_of_many_parts(ba, shape, groups, layout):
    """Units whose partials come from many CTAs: the same bits from launches
    that find the caches cold and from ones that do not, and the definition's
    statistics each time."""
    junk = torch.empty(48 << 20, device="cuda")
    x = _x(shape, torch.float32, layout, offset=2.0)
    r = x.double().reshape(shape[0], groups, -1)
    ref = (r - r.mean(-1, keepdim=True)) / torch.sqrt(r.var(-1, correction=0, keepdim=True) + 1e-5)
    ref = ref.reshape(shape)
    first = ba.ops.group_norm(x, groups)
    # as K above: 160 u R rstd, R rstd below 8 here, plus 4 u M rstd
    assert float((first.double() - ref).abs().max()) <= 160 * U * 8 + 4 * U * 16 + 160 * U * 8
    for i in range(40):
        if i % 2:
            junk.zero_()
        assert torch.equal(ba.ops.group_norm(x, groups), first)
    from batchaug_b200 import _lib as L
    L.wait_status(x.device)
