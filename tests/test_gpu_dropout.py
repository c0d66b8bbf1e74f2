"""Counter-based dropout (ba_dropout) against its definition in 64 bits.

Which voxels stay is compared exactly.  What stays is x * scale, rounded once
to the tensor's type, with scale = 1 / (1 - p) rounded to fp32: two fp32
roundings of half a step and, for bf16, one of half a bf16 step, each
relative to the value."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import feature_ref as R

pytestmark = pytest.mark.gpu

# relative: eps/2 of the stored type, and two half steps of fp32
TOL = {torch.float32: 2 * 2.0**-24 + 2.0**-24, torch.bfloat16: 2.0**-8 + 2 * 2.0**-24}


def _x(shape, dtype, layout, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g).to(dtype)
    x = x + (x == 0)  # no zeros: what is zero in the result was dropped
    x = x.cuda()
    return x.contiguous(memory_format=torch.channels_last_3d) if layout == "last" else x


def _check(y, x, f, tol=None):
    assert y.dtype == x.dtype and y.shape == x.shape and y.stride() == x.stride()
    y64, ref = y.detach().double().cpu(), x.detach().double().cpu() * f
    assert torch.equal(y64 != 0, f != 0)
    assert ((y64 - ref).abs() <= (tol or TOL[x.dtype]) * ref.abs()).all()


SHAPES = [
    (1, 1, 1, 1, 1), (2, 3, 1, 1, 7), (1, 8, 2, 2, 2), (2, 16, 3, 5, 7), (1, 4, 8, 8, 9),
    (2, 12, 5, 4, 4), (3, 33, 3, 3, 3), (1, 2, 9, 16, 32), (1, 5, 17, 19, 23), (1, 2056, 1, 2, 5),
    (2, 520, 2, 3, 3), (1, 1, 20, 20, 20), (2, 20, 1, 3, 43),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("shape", SHAPES)
def test_bits_and_values(ba, shape, layout, dtype):
    x = _x(shape, dtype, layout)
    for p, seed in ((0.3, 12345), (0.5, 2**63 + 11)):
        y = ba.ops.dropout(x, p, seed, elem_offset=2**32 + 5)
        _check(y, x, R.factor(shape, p, seed, 2**32 + 5))
    y = ba.ops.dropout(x, 0.4, 9, channelwise=True, rescale=False)
    _check(y, x, R.factor(shape, 0.4, 9, channelwise=True, rescale=False), tol=0.0)


@pytest.mark.parametrize("p", [0.0, 1.0, 2.0**-32, 2.0**-16, 1 - 2.0**-16, 1 - 2.0**-24, 0.25,
                               1.00001 * 2.0**-16])
def test_rates_at_the_threshold(ba, p):
    """Thresholds whose halves are zero, full, or met by a voxel's."""
    shape = (1, 8, 16, 16, 32)
    x = _x(shape, torch.float32, "last")
    y = ba.ops.dropout(x, p, 77)
    _check(y, x, R.factor(shape, p, 77))


def test_low_halves_decide(ba):
    """Thresholds put on and just above the number of a voxel: the high halves
    tie and the low halves decide (numbers a float's 24 bits can hold)."""
    shape = (1, 2, 4, 8, 64)
    r = R.numbers(1, 2, 2048, 31).reshape(-1)
    small = [int(v) for v in r if v < 2**24 and v & 0xFFFF][:4]
    assert small, "the seed gives no small numbers"
    x = _x(shape, torch.float32, "first")
    for v in small:
        for t, kept in ((v, True), (v + 1, False)):
            y = ba.ops.dropout(x, t / 2.0**32, 31)
            f = R.factor(shape, t / 2.0**32, 31)
            assert bool(f.reshape(-1)[int(np.flatnonzero(r == v)[0])] != 0) == kept
            _check(y, x, f)


def test_rate_of_each_element_and_mask(ba):
    shape = (5, 6, 7, 5, 3)
    p = torch.tensor([0.0, 1.0, 0.3, 0.9, float("nan")], device="cuda")
    mask = torch.tensor([True, True, True, False, True], device="cuda")
    for layout in ("first", "last"):
        x = _x(shape, torch.bfloat16, layout)
        f = R.factor(shape, p.cpu().numpy(), 3, mask=mask.cpu().numpy())
        _check(ba.ops.dropout(x, p, 3, mask=mask), x, f)
        _check(ba.ops.dropout(x, p, 3, mask=mask.cpu().numpy()), x, f)
    # rates outside [0, 1] in a tensor are clamped
    q = torch.tensor([-1.0, 2.0, 0.0, 1.0, -0.0], device="cuda")
    x = _x(shape, torch.float32, "first")
    _check(ba.ops.dropout(x, q, 3), x, R.factor(shape, [0, 1, 0, 1, 0], 3))


def test_layout_and_sharding_keep_the_bits(ba):
    shape = (4, 24, 5, 6, 7)
    first, last = _x(shape, torch.float32, "first"), _x(shape, torch.float32, "last")
    a, b = ba.ops.dropout(first, 0.2, 8), ba.ops.dropout(last, 0.2, 8)
    assert torch.equal(a, b)
    part = ba.ops.dropout(first[2:], 0.2, 8, elem_offset=2)
    assert torch.equal(a[2:], part)
    assert not torch.equal(a, ba.ops.dropout(first, 0.2, 9))
    assert torch.equal(a, ba.ops.dropout(first, 0.2, 8 + 2**64))  # keys are 64 bits


def test_dropped_values_are_zero_whatever_they_were(ba):
    shape = (1, 4, 8, 8, 8)
    f = R.factor(shape, 0.5, 4)
    for bad in (float("nan"), float("inf")):
        x = torch.full(shape, bad, device="cuda")
        y = ba.ops.dropout(x, 0.5, 4)
        assert torch.equal(y.cpu() == 0, f == 0)


def test_views_and_unaligned_storage(ba):
    base = _x((1, 1, 1, 1, 8 * 6 * 4 * 4 * 4 + 1), torch.bfloat16, "first").reshape(-1)
    x = base[1:].view(8, 6, 4, 4, 4)  # 2 bytes past a 16-byte boundary
    _check(ba.ops.dropout(x, 0.3, 2), x, R.factor(x.shape, 0.3, 2))
    v = _x((2, 8, 6, 6, 6), torch.float32, "first")[:, 1:7:2, ::2]  # neither layout: copied
    y = ba.ops.dropout(v, 0.3, 2)
    _check(y, v.contiguous(), R.factor(v.shape, 0.3, 2))


@pytest.mark.parametrize("layout", ["first", "last"])
def test_gradient(ba, layout):
    shape = (2, 12, 5, 6, 7)
    x = _x(shape, torch.float32, layout).requires_grad_()
    dy = _x(shape, torch.float32, "first", seed=1)
    mask = torch.tensor([True, False], device="cuda")
    y = ba.ops.dropout(x, 0.25, 6, mask=mask)
    f = R.factor(shape, 0.25, 6, mask=mask.cpu().numpy())
    _check(y.detach(), x.detach(), f)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx.stride() == x.stride()
    _check(dx, dy if layout == "first" else dy.to(memory_format=torch.channels_last_3d), f)
    # a broadcast gradient
    (dx,) = torch.autograd.grad(ba.ops.dropout(x, 0.25, 6, mask=mask).sum(), x)
    _check(dx, torch.ones_like(x), f)


def test_empty(ba):
    for shape in ((0, 3, 2, 2, 2), (2, 0, 2, 2, 2), (2, 3, 0, 2, 2)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = ba.ops.dropout(x, 0.5, 1)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape


def test_seed_in_device_memory_and_graph(ba):
    """A captured graph reads the seed when it is replayed."""
    shape = (2, 16, 6, 6, 6)
    x = _x(shape, torch.float32, "last")
    seed = torch.tensor([41], dtype=torch.int64, device="cuda")
    assert torch.equal(ba.ops.dropout(x, 0.3, seed), ba.ops.dropout(x, 0.3, 41))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ba.ops.dropout(x, 0.3, seed)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ba.ops.dropout(x, 0.3, seed)
        seed.add_(1)
    seed.fill_(100)
    for s in (100, 101):
        g.replay()
        _check(y, x, R.factor(shape, 0.3, s))
    neg = torch.tensor([-3], dtype=torch.int64, device="cuda")
    _check(ba.ops.dropout(x, 0.3, neg), x, R.factor(shape, 0.3, 2**64 - 3))


def test_refusals(ba):
    x = torch.zeros(2, 3, 4, 4, 4, device="cuda")
    ops = ba.ops
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            ops.dropout(x, bad, 1)
    with pytest.raises(ValueError, match="values for a batch"):
        ops.dropout(x, torch.zeros(3, device="cuda"), 1)
    with pytest.raises(ValueError, match="seed"):
        ops.dropout(x, 0.5, None)
    with pytest.raises(ValueError, match="seed tensor"):
        ops.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="seed tensor"):
        ops.dropout(x, 0.5, torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="B,C,H,W,D"):
        ops.dropout(x[0], 0.5, 1)
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        ops.dropout(x.half(), 0.5, 1)
