"""Dropout and group norm where a program may take them without thinking of
them: saved tensors that come back elsewhere, a graph walked twice, some of the
gradients only, a first call under capture, launches side by side, offsets past
32 bits, a great many small units.  Tolerances are test_gpu_group_norm's."""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys

import pytest
import torch
import torch.utils.checkpoint

import feature_ref as R
import test_gpu_group_norm as N

pytestmark = pytest.mark.gpu


def _leaves(x, kind=torch.float32):
    w, b = N._params(x.shape[1], kind)
    return [t.detach().clone(memory_format=torch.preserve_format).requires_grad_()
            for t in (x, w, b)]


@pytest.mark.parametrize("layout", ["first", "last"])
def test_saved_tensors_that_come_back_elsewhere(ba, layout):
    """Offloading moves what the backward pass reads, and drops its strides;
    recomputation frees it in between."""
    x = N._x((2, 16, 6, 7, 8), torch.float32, layout)
    leaves = _leaves(x)
    dy = N._x((2, 16, 6, 7, 8), torch.float32, layout, seed=1)

    def run(x, w, b):  # an input of the operator's own, free once nothing saves it
        y = ba.ops.group_norm(x * 1.0, 4, w, b, activation="silu", p=0.3, seed=5)
        return ba.ops.dropout(y, torch.tensor([0.2, 0.4], device="cuda"), 6)

    want = torch.autograd.grad(run(*leaves), leaves, dy)

    def offload(pin):
        with torch.autograd.graph.save_on_cpu(pin_memory=pin):
            y = run(*leaves)
        junk = [torch.full_like(x, float("nan")) for _ in range(8)]  # over what was freed
        got = torch.autograd.grad(y, leaves, dy)
        del junk
        return got

    def recompute():
        y = torch.utils.checkpoint.checkpoint(run, *leaves, use_reentrant=False)
        junk = [torch.full_like(x, float("nan")) for _ in range(8)]
        got = torch.autograd.grad(y, leaves, dy)
        del junk
        return got

    for got in (offload(False), offload(True), recompute()):
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_a_graph_walked_twice_and_parts_of_it(ba):
    x, w, b = _leaves(N._x((2, 8, 9, 10, 11), torch.bfloat16, "last"))
    dy = N._x((2, 8, 9, 10, 11), torch.bfloat16, "last", seed=2)
    y = ba.ops.group_norm(x, 2, w, b, activation="gelu", p=0.1, seed=1)
    full = torch.autograd.grad(y, [x, w, b], dy, retain_graph=True)
    again = torch.autograd.grad(y, [x, w, b], dy, retain_graph=True)
    assert all(torch.equal(a, c) for a, c in zip(full, again))
    # some leaves only: dx not computed, or no parameters' gradients
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        y = ba.ops.group_norm(leaves[0], 2, *leaves[1:], activation="gelu", p=0.1, seed=1)
        (g,) = torch.autograd.grad(y, leaves[i], dy)
        assert torch.equal(g, full[i])


def test_rates_of_elements_and_a_seed_on_the_device(ba):
    x = N._x((3, 8, 5, 6, 7), torch.float32, "last")
    rates = torch.tensor([0.0, 1.0, 0.35], device="cuda")
    seed = torch.tensor([-3], dtype=torch.int64, device="cuda")
    dy = N._x((3, 8, 5, 6, 7), torch.float32, "last", seed=4)
    a, c = (x.clone(memory_format=torch.preserve_format).requires_grad_() for _ in range(2))
    y = ba.ops.group_norm(a, 2, activation="silu", p=rates, seed=seed, elem_offset=2**32 + 5)
    z = ba.ops.dropout(ba.ops.group_norm(c, 2, activation="silu"), rates, -3,
                       elem_offset=2**32 + 5)
    assert torch.equal(y, z)
    assert not y[1].any()
    ga, gc = torch.autograd.grad(y, a, dy)[0], torch.autograd.grad(z, c, dy)[0]
    # dy scaled before or after one fp32 product: a few units of the terms
    assert (ga - gc).abs().max() <= 64 * N.U * gc.abs().max()


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("shape, groups", [((5000, 16, 1, 2, 3), 4), ((700, 24, 4, 4, 4), 24)])
def test_many_small_units(ba, shape, groups, layout):
    N._run(ba, shape, torch.float32, layout, groups, "silu")


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("shape, groups", [((1, 8, 40, 44, 48), 1), ((2, 6, 47, 53, 37), 2)])
def test_units_of_many_thread_blocks(ba, shape, groups, p, dtype, layout):
    """Above what a cluster takes: waiting launches, pieces of the results."""
    N._run(ba, shape, dtype, layout, groups, "silu", p=p)


@pytest.mark.parametrize("layout", ["first", "last"])
def test_several_waves(ba, layout):
    """85 MB of units in two waves and more, forward and backward, as the same
    elements on their own.  |x - mean|, |xh| and |dy| are below 8 and rstd about 1,
    so K is below 2e-4, dz within 8 (K + 16 u 9) < 2e-3, and dx, with the two
    means' errors on top, within 2e-3 (1 + 1 + 8 8) < 0.14 of a value that a wrong
    place would change by whole units; on average the errors are 2e-3 at most."""
    shape = (6, 4, 96, 96, 96)
    x = N._x(shape, torch.float32, layout).requires_grad_()
    dy = N._x(shape, torch.float32, layout, seed=3)
    y = ba.ops.group_norm(x, 4 if layout == "first" else 2, activation="silu", p=0.1, seed=2)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert float(dy.abs().max()) < 8
    for b in range(6):
        one = x.detach()[b:b + 1].clone(memory_format=torch.preserve_format).requires_grad_()
        z = ba.ops.group_norm(one, 4 if layout == "first" else 2, activation="silu", p=0.1, seed=2,
                              elem_offset=b)
        (dz,) = torch.autograd.grad(z, one, dy[b:b + 1])
        assert (y[b] - z[0]).abs().max() <= 2 * 1.2 * 1.13 * 2e-4
        e = (dx[b] - dz[0]).abs()
        assert e.max() <= 0.28 and e.mean() <= 4e-3


@pytest.mark.parametrize("dtype, shape, groups", [
    (torch.bfloat16, (2, 2056, 1, 3, 3), 257), (torch.float32, (2, 1028, 2, 2, 3), 257),
    (torch.bfloat16, (1, 8200, 1, 1, 3), 8), (torch.float32, (1, 1542, 1, 2, 2), 6)])
def test_groups_that_begin_in_a_later_pass(ba, dtype, shape, groups):
    """Rows wider than a pass of a thread block (256 accesses)."""
    N._run(ba, shape, dtype, "last", groups, "silu")


@pytest.mark.parametrize("layout", ["first", "last"])
def test_launches_side_by_side(ba, layout):
    """Launches that fill the device and wait within themselves, from three
    streams, with dropouts between them."""
    from batchaug_b200 import _lib as L
    x = N._x((2, 32, 48, 48, 48), torch.bfloat16, layout)
    leaves = _leaves(x)

    def step():
        y = ba.ops.group_norm(leaves[0], 8, *leaves[1:], activation="silu")
        y = ba.ops.dropout(y, 0.25, 9)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, x))

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, c) for a, c in zip(g, want))
    L.wait_status(x.device)


def test_first_call_is_captured(ba):
    """Nothing of the library has run in the process before."""
    code = """
import torch, batchaug_b200 as ba
x = torch.randn(2, 16, 40, 40, 40, device='cuda')
s = torch.randn(2, 16, 4, 4, 4, device='cuda').contiguous(memory_format=torch.channels_last_3d)
def step():
    return (ba.group_norm(x, 4, activation='silu', p=0.2, seed=3), ba.dropout(x, 0.5, 4),
            ba.group_norm(s, 4), ba.group_norm(s.repeat(1, 1, 9, 9, 9), 4))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
for _ in range(2):
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=root + os.pathsep + os.environ.get("PYTHONPATH", ""))
    r = subprocess.run([sys.executable, "-c", code], env=env, cwd=root, timeout=120,
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("layout", ["first", "last"])
def test_offsets_past_32_bits(ba, layout):
    """2.3e9 values: the last element as on its own."""
    shape = (5, 8, 384, 384, 384)
    fmt = torch.channels_last_3d if layout == "last" else torch.contiguous_format
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda", memory_format=fmt).normal_()
    tail = x[4:].clone(memory_format=torch.preserve_format)
    y = ba.ops.dropout(x, 0.3, 8)
    assert torch.equal(y[4:], ba.ops.dropout(tail, 0.3, 8, elem_offset=4))
    del y
    y = ba.ops.group_norm(x, 2)[4:].float()
    ref = ba.ops.group_norm(tail, 2).float()
    # either is within K (R and M below 8, rstd about 1) and a half step of the truth
    K = 160 * N.U * 8 + 4 * N.U * 8 + 160 * N.U * 8
    y -= ref
    assert (y.abs_() <= 2 * K + 2 * N._half_step(torch.bfloat16) * (ref.abs_() + K)).all()


@pytest.mark.parametrize("op", ["norm", "dropout"])
def test_derivatives_that_would_be_lost_are_refused(ba, op):
    """Forward mode over the call or over its gradient, and a recorded call; a
    dual level without tangents, and a program compiled around the call, go on."""
    fwd = torch.autograd.forward_ad

    def f(t):
        if op == "norm":
            return ba.ops.group_norm(t, 2, activation="silu")
        return ba.ops.dropout(t, 0.5, 3)

    x = N._x((2, 8, 4, 5, 6), torch.float32, "last")
    leaf = x.clone(memory_format=torch.preserve_format).requires_grad_()
    y = f(leaf)
    with fwd.dual_level():
        one = torch.ones_like(x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(fwd.make_dual(x, one))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(fwd.make_dual(leaf, one))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaf, fwd.make_dual(one, one), retain_graph=True)
        assert torch.equal(f(x), y)
        torch.autograd.grad(y, leaf, one, retain_graph=True)
    with pytest.raises(NotImplementedError, match="recorded"):
        torch.jit.trace(f, (x,))
    compiled = torch.compile(lambda t: f(t * 2.0) + 1.0, backend="eager")
    assert torch.equal(compiled(x), f(x * 2.0) + 1.0)


def _part_of_a_thread_block(x, groups, layout):
    """Voxels of a thread block's (channels last) or a warp's part of the sums
    of a single unit, from the size of the scratch: 16 bytes, 16 more with
    pieces of results (channels first), and 16 for each part."""
    from batchaug_b200 import _lib as L
    B, C, H, W, D = x.shape
    assert B == groups == 1
    last = layout == "last"
    desc = L.norm_desc(x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, B, C, H, W, D, groups, L.BA_F32,
                       L.BA_CHANNELS_LAST if last else L.BA_CHANNELS_FIRST, L.BA_F32,
                       L.BA_ACT_NONE, 1e-5, 0.0, 0.0, 0, 0, 0, 0, 0)
    n = L.lib.ba_norm_workspace_bytes(ctypes.byref(desc), 0) // 16 - (1 if last else 2)
    parts, grain = (n, 8) if last else (n * 8 // C, 256)
    return -(-(-(-H * W * D // parts)) // grain) * grain


@pytest.mark.parametrize("layout, shape", [("last", (1, 512, 64, 64, 64)),
                                           ("first", (1, 32, 128, 128, 128))])
@pytest.mark.parametrize("noise", [0.0, 1.0])
def test_variance_where_every_thread_begins_with_background(ba, layout, shape, noise):
    """About 300 (last) and 600 values a thread, its first ones 0 and the others
    1001.3 or so: sums about a thread's first value would be off by so many times
    their own errors.  With u = 2^-24: m values summed in fp32 about a centre of theirs have
    an M2 within A (3 m + 2) u of itself, where A is the sum of squares over M2,
    for the roundings of the sum, of the squares and of the first moment.  A
    thread's first 8 values have m = 8 and A <= 8 (208 u; channels first 4
    accumulators of 8 and an A of 32 / 4), later sums m <= 32 and A <= 2 (196 u),
    each centre one u more (20 at most), and eight threads that meet 8 (3 8 + 2) u:
    the variance within 440 u, and z within 220 u |z|, 4 u |z| for its own
    roundings, plus test_gpu_group_norm's bound for the mean."""
    x = torch.full(shape, 1001.3, device="cuda")
    if noise:
        x += noise * torch.randn(shape, generator=torch.Generator("cuda").manual_seed(1),
                                 device="cuda")
    if layout == "last":
        x = x.contiguous(memory_format=torch.channels_last_3d)
    S = shape[2] * shape[3] * shape[4]
    part = _part_of_a_thread_block(x, 1, layout)
    assert 400 * (2 if layout == "last" else 32) < part < 800 * (2 if layout == "last" else 32)
    first = (torch.arange(S, device="cuda") % part) < (2 if layout == "last" else 128)
    x.masked_fill_(first.view(1, 1, *shape[2:]), 0.0)
    mean = x.double().mean()
    d = x.double().sub_(mean)
    rstd = 1 / torch.sqrt(d.square().mean() + 1e-5)
    R, M = float(d.abs().max()), float(x.max())
    z = d.mul_(rstd)
    tol = float(rstd) * (160 * N.U * R + 4 * N.U * M) + 224 * N.U * z.abs()
    y = ba.ops.group_norm(x, 1)
    err = (y.double() - z).abs_().div_(tol)
    assert float(err.max()) <= 1, float(err.max())


def _line(ba, z_lo, z_hi, dtype, act, layout, n=1 << 16):
    """(z, act(z)) along a line: x = z in that type, its mean and deviation put
    back by bias and weight; z as the operator itself has it, unrounded in fp32."""
    x = torch.linspace(z_lo, z_hi, n, device="cuda").to(dtype)
    v = x.double()
    w, b = ((t.float() * torch.ones(1 if layout == "first" else n, device="cuda"))
            for t in (v.var(correction=0).sqrt(), v.mean()))
    x = x.view(1, 1, n, 1, 1) if layout == "first" else x.view(1, n, 1, 1, 1)
    if layout == "last":
        x = x.contiguous(memory_format=torch.channels_last_3d)
    z = ba.ops.group_norm(x.float(), 1, w, b, eps=0.0)
    y = ba.ops.group_norm(x, 1, w, b, eps=0.0, activation=act)
    return z.flatten().double(), y.flatten().double()


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gelu_keeps_the_digits_of_its_tail(ba, dtype, layout):
    """With u = 2^-24: the tail's fit is within 2.8 u of its value (bf16: 78 u) and
    its sum of products 6 u more, the reciprocal within 2 u, the exponential 4 u,
    its argument (fp32: given back; bf16: z^2 u) and the last products 3 u: y
    within 24 u (bf16: 100 u + z^2 u) of itself, and then a half step."""
    z, y = _line(ba, -12.0, 12.0, dtype, "gelu", layout)
    ref = z * 0.5 * torch.special.erfc(-z / 2**0.5)
    rel = 24 * N.U if dtype == torch.float32 else (100 + z * z) * N.U + N._half_step(dtype)
    err = (y - ref).abs() / (rel * ref.abs()).clamp(min=2.0**-126)
    assert float(err.max()) <= 1, (float(err.max()), float(z[err.argmax()]))


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_silu_far_below_zero(ba, dtype, layout):
    """With u = 2^-24: the exponential within 4 u, its argument (fp32: given back, 2
    u; bf16: |z| u), the sum 1 u, the reciprocal 2 u, the product 1 u, and then
    a half step.  exp(80) is 5e34, so nothing leaves the range of fp32."""
    z, y = _line(ba, -80.0, 80.0, dtype, "silu", layout)
    ref = z / (1 + torch.exp(-z))
    rel = 10 * N.U if dtype == torch.float32 else (8 + z.abs()) * N.U + N._half_step(dtype)
    err = (y - ref).abs() / (rel * ref.abs()).clamp(min=2.0**-126)
    assert float(err.max()) <= 1, (float(err.max()), float(z[err.argmax()]))


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "leaky_relu"])
def test_activations_of_the_largest_values(ba, act, dtype, layout):
    """A weight that takes z to the end of the type's range and past it: the far
    ends of the activations are z (or infinity) and 0 (leaky: a hundredth)."""
    x = N._x((1, 2, 4, 4, 4), dtype, layout)
    y = ba.ops.group_norm(x, 1, torch.tensor([3e38, 1e20], device="cuda"), activation=act).double()
    z = ba.ops.group_norm(x, 1, torch.tensor([3e38, 1e20], device="cuda")).double()
    assert bool(torch.isinf(z).any())
    up = z > 0
    assert torch.equal(y[up], z[up])
    low = y[~up & torch.isfinite(z)]
    if act == "leaky_relu":
        ref = 0.01 * z[~up & torch.isfinite(z)]
        # the slope's and the product's roundings, and the type's on both sides
        assert ((low - ref).abs() <= (4 * N.U + 2.1 * N._half_step(dtype)) * ref.abs()).all()
    else:
        assert not low.any()


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape, groups", [((2, 16, 6, 7, 8), 4), ((2, 6, 5, 5, 5), 3)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rectified_values_stop_any_gradient(ba, bad, shape, groups, dtype, layout):
    """An infinite or undefined gradient of a value that the rectifier has put to
    zero counts as none, as in torch; one of a dropped value too."""
    for p in (0.0, 0.4):
        leaves = _leaves(N._x(shape, dtype, layout))
        y = ba.ops.group_norm(leaves[0], groups, *leaves[1:], activation="relu", p=p, seed=3)
        dy = N._x(shape, dtype, layout, seed=1)
        dead = y.detach() == 0
        assert bool(dead.any())
        clean = torch.autograd.grad(y, leaves, dy.masked_fill(dead, 0.0), retain_graph=True)
        got = torch.autograd.grad(y, leaves, dy.masked_fill(dead, bad))
        assert all(torch.equal(a, c) for a, c in zip(got, clean))


@pytest.mark.parametrize("layout", ["first", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 16, 8, 24, 20), (2, 3, 31, 33, 35), (3, 20, 9, 11, 13)])
@pytest.mark.parametrize("flags", [0, 1, 2])
def test_dropout_in_place(ba, shape, dtype, layout, flags):
    """The C entry with dst == src (the Python function has a result of its own),
    in a captured graph too: the second replay drops from what the first left."""
    from batchaug_b200 import _lib as L
    x = N._x(shape, dtype, layout)
    B, C, H, W, D = shape
    want = [ba.ops.dropout(x, 0.4, 7, channelwise=bool(flags & 1), rescale=bool(flags & 2))]
    want.append(ba.ops.dropout(want[0], 0.4, 7, channelwise=bool(flags & 1),
                               rescale=bool(flags & 2)))
    v = x.clone(memory_format=torch.preserve_format)
    d = L.dropout_desc(v.data_ptr(), v.data_ptr(), B, C, H, W, D, L.dtype_code(x),
                       L.BA_CHANNELS_LAST if layout == "last" else L.BA_CHANNELS_FIRST, flags,
                       0.4, 0, 0, 7, 0, 0)
    L.check(L.lib.ba_dropout(ctypes.byref(d), L.stream_ptr(x.device)), "ba_dropout")
    assert torch.equal(v, want[0])
    v.copy_(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.check(L.lib.ba_dropout(ctypes.byref(d), L.stream_ptr(x.device)), "ba_dropout")
    for w in want:
        g.replay()
        assert torch.equal(v, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape, groups", [
    ((1, 128, 10, 10, 10), 1), ((2, 72, 8, 8, 9), 1), ((2, 256, 6, 6, 7), 2),
    ((20, 256, 4, 4, 4), 8), ((40, 64, 4, 4, 4), 1)])
def test_groups_of_many_channels(ba, shape, groups, dtype):
    """Channels first, more channels to a group than a cluster has warps, or as
    many clusters as do not fit the device at once."""
    N._run(ba, shape, dtype, "first", groups, "silu")


@pytest.mark.parametrize("layout", ["first", "last"])
def test_several_waves_against_the_definition(ba, layout):
    """The 85 MB of test_several_waves in 64 bits on the device, every value
    within test_gpu_group_norm's bounds (a thread sums 64 values or fewer here)."""
    shape, groups = (6, 4, 96, 96, 96), 4 if layout == "first" else 2
    x = N._x(shape, torch.float32, layout).requires_grad_()
    dy = N._x(shape, torch.float32, layout, seed=3)
    y = ba.ops.group_norm(x, groups, activation="silu")
    (dx,) = torch.autograd.grad(y, x, dy)
    for b in range(shape[0]):
        one = x.detach()[b:b + 1].double().contiguous().requires_grad_()
        g = dy[b:b + 1].double()
        ref, z = R.norm(one, groups, act="silu")
        (ref_dx,) = torch.autograd.grad(ref, one, g)
        ref, z = ref.detach(), z.detach()
        K, rstd = N._bounds(one.detach(), groups, None, 1e-5, z)
        tol = 1.13 * K + 16 * N.U * (ref.abs() + z.abs() + 1) + N._half_step(y.dtype) * ref.abs()
        assert ((y.detach()[b:b + 1].double() - ref).abs() <= tol).all()
        s = torch.sigmoid(z)
        dz = g * (s + z * s * (1 - s))
        e_dz = g.abs() * (K + 16 * N.U * (1 + z.abs()))
        t1, t2 = dz.abs(), (dz * z).abs()
        e1, e2 = e_dz + 80 * N.U * t1, e_dz * z.abs() + t1 * K + 80 * N.U * t2
        m = {k: N._gmean(t, groups) for k, t in (("e1", e1), ("e2", e2), ("t1", t1), ("t2", t2))}
        tol = rstd * (e_dz + m["e1"] + z.abs() * m["e2"] + K * m["t2"]
                      + 176 * N.U * (t1 + m["t1"] + z.abs() * m["t2"])) \
            + N._half_step(dx.dtype) * ref_dx.abs()
        assert float(tol.mean()) < 1e-3
        assert ((dx[b:b + 1].double() - ref_dx).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 6, 3, 6, 10), (1, 4, 2, 2, 33), (2, 8, 2, 9, 14)])
def test_channels_that_end_within_a_dropout_block(ba, shape, dtype):
    """Channels first, lengths of 8 k + 4: whole 16-byte accesses in fp32, the last
    of them half a block of the generator."""
    assert (shape[2] * shape[3] * shape[4]) % 8 == 4
    N._run(ba, shape, dtype, "first", 2, "silu", p=0.3, seed=2**33 + 7)
    x = N._x(shape, dtype, "first")
    f = R.factor(shape, 0.3, 11).cuda()
    y = ba.ops.dropout(x, 0.3, 11)
    assert torch.equal(y == 0, f == 0)
    ref = x.double() * f
    # 1 - p, the reciprocal, the product, then the type's half step
    assert ((y.double() - ref).abs() <= (4 * N.U + N._half_step(dtype)) * ref.abs()).all()
