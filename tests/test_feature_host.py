"""Group norm and dropout without a GPU: refusals of the C ABI and of the
functions, scratch sizes, struct layouts."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import feature_ref as R
from conftest import ROOT


def _drop(L, **kw):
    d = L.DropoutDesc(4096, 8192, 2, 3, 4, 4, 4, L.BA_F32, L.BA_CHANNELS_FIRST,
                      L.BA_DROPOUT_RESCALE, 0.5)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _norm(L, **kw):
    # made-up addresses: every call here is refused before a launch
    d = L.NormDesc(x=1 << 20, dy=1 << 21, out=1 << 22, stats=1 << 23, batch=2, channels=6, H=4,
                   W=4, D=4, groups=3, dtype=L.BA_F32, layout=L.BA_CHANNELS_LAST, eps=1e-5)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_struct_layouts_match_header(ba, tmp_path):
    from batchaug_b200 import _lib as L
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = {"ba_dropout_desc": L.DropoutDesc, "ba_norm_desc": L.NormDesc}
    lines = ['#include <stdio.h>', '#include "batchaug_b200.h"', "int main(void) {"]
    for cname, ct in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in ct._fields_:
            lines.append(f'printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    exe = tmp_path / "probe"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    lines = [line.split() for line in got if line]
    assert len(lines) == sum(len(c._fields_) + 1 for c in structs.values())
    for cname, what, val in lines:
        ct = structs[cname]
        assert int(val) == (ctypes.sizeof(ct) if what == "size" else getattr(ct, what).offset)


@pytest.mark.parametrize("kw, word", [
    (dict(dtype=7), b"dtype"), (dict(layout=2), b"layout"), (dict(flags=8), b"flags"),
    (dict(p=1.5), b"p="), (dict(p=float("nan")), b"p="), (dict(batch=-1), b"negative"),
    (dict(src=None), b"NULL"), (dict(dst=None), b"NULL"), (dict(src=4098), b"aligned"),
    (dict(dst=4096 + 64), b"overlaps"), (dict(p_elem=2), b"aligned"), (dict(seed_dev=4), b"aligned"),
    (dict(H=1 << 30, W=1 << 30), b"2^40"), (dict(batch=1 << 31, channels=1, H=1, W=1, D=1), b"2^31"),
])
def test_dropout_refusals(ba, kw, word):
    from batchaug_b200 import _lib as L
    assert L.lib.ba_dropout(ctypes.byref(_drop(L, **kw)), None) == L.BA_EINVAL
    assert word in L.lib.ba_last_error()
    assert L.lib.ba_dropout(None, None) == L.BA_EINVAL


@pytest.mark.parametrize("kw, word", [
    (dict(dtype=7), b"dtype"), (dict(layout=2), b"layout"), (dict(groups=0), b"groups"),
    (dict(groups=4), b"divide"), (dict(param_dtype=3), b"param_dtype"),
    (dict(activation=9), b"activation"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(p=-0.5), b"p="), (dict(x=None), b"NULL"), (dict(stats=None), b"NULL"),
    (dict(x=(1 << 20) + 2), b"aligned"), (dict(stats=(1 << 23) + 4), b"aligned"),
    (dict(weight=2), b"aligned"), (dict(out=(1 << 20) + 16), b"overlaps"),
    (dict(batch=1 << 30, channels=6, groups=6, H=1, W=1, D=1), b"2^31"),
])
@pytest.mark.parametrize("backward", [False, True])
def test_norm_refusals(ba, kw, word, backward):
    from batchaug_b200 import _lib as L
    fn = L.lib.ba_norm_backward if backward else L.lib.ba_norm_forward
    assert fn(ctypes.byref(_norm(L, **kw)), 1 << 24, 1 << 30, None) == L.BA_EINVAL
    assert word in L.lib.ba_last_error()
    assert fn(None, None, 0, None) == L.BA_EINVAL


def test_norm_scratch_is_checked(ba):
    from batchaug_b200 import _lib as L
    d = _norm(L)
    for backward, fn in ((0, L.lib.ba_norm_forward), (1, L.lib.ba_norm_backward)):
        size = L.lib.ba_norm_workspace_bytes(ctypes.byref(d), backward)
        assert size > 0
        assert fn(ctypes.byref(d), 1 << 24, size - 1, None) == L.BA_EINVAL
        assert b"workspace" in L.lib.ba_last_error()
        assert fn(ctypes.byref(d), (1 << 24) + 8, size, None) == L.BA_EINVAL
        assert b"aligned" in L.lib.ba_last_error()
    assert L.lib.ba_norm_workspace_bytes(ctypes.byref(_norm(L, groups=4)), 0) == 0
    assert L.lib.ba_norm_workspace_bytes(ctypes.byref(_norm(L, D=0)), 0) == 0
    # the backward pass alone reads dy
    d = _norm(L, dy=None)
    assert L.lib.ba_norm_backward(ctypes.byref(d), 1 << 24, 1 << 30, None) == L.BA_EINVAL
    # nothing to do
    for fn in (L.lib.ba_norm_forward, L.lib.ba_norm_backward):
        assert fn(ctypes.byref(_norm(L, batch=0, x=None, out=None)), None, 0, None) == L.BA_OK
    assert L.lib.ba_dropout(ctypes.byref(_drop(L, W=0, src=None)), None) == L.BA_OK


def test_functions_want_cuda_tensors(ba):
    from batchaug_b200 import ops
    x = torch.zeros(2, 4, 3, 3, 3)
    with pytest.raises(ValueError, match="CUDA"):
        ops.group_norm(x, 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.dropout(x, 0.5, 1)


def test_reference_bits_known_answer():
    """The tests' own generator against Random123's published vectors."""
    w = R.philox(0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344, 0x299F31D0A4093822)
    assert [int(v) for v in w] == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    r = R.numbers(2, 3, 1000, 5)
    assert abs(r.mean() / 2**32 - 0.5) < 0.02 and len(np.unique(r)) == r.size


def test_dropout_op_of_a_chain(ba):
    from batchaug_b200 import _lib as L
    c = L.ChainDesc()
    c.batch, c.channels, c.H, c.W, c.D, c.dtype, c.n_ops = 1, 1, 2, 2, 2, 0, 1
    c.ops[0].kind = L.BA_OP_DROPOUT
    assert L.lib.ba_intensity_chain(ctypes.byref(c), None, 0, None) == L.BA_EINVAL
    assert b"rate" in L.lib.ba_last_error()
    c.ops[0].param, c.ops[0].flags = 8, 4
    assert L.lib.ba_intensity_chain(ctypes.byref(c), None, 0, None) == L.BA_EINVAL
    assert b"flags" in L.lib.ba_last_error()
    c.ops[0].kind = L.BA_OP_DROPOUT + 1
    assert L.lib.ba_intensity_chain(ctypes.byref(c), None, 0, None) == L.BA_EINVAL
    assert b"unknown kind" in L.lib.ba_last_error()


def test_transform_params_on_the_host(ba):
    """The dropout transform's draws are keyed on the global element, and its
    chain op carries seed, offset and flags."""
    from batchaug_b200 import _lib as L
    t = ba.RandVoxelDropout(prob=0.5, rate=(0.1, 0.3), channel_wise=True)
    torch.manual_seed(1)
    whole = t.sample_host(6, (6, 2, 4, 4, 4))
    torch.manual_seed(1)
    with ba.shard(4, 6):
        p = t.sample_params(2, (2, 2, 4, 4, 4), torch.device("cpu"))
    part = p["_host"]
    assert np.array_equal(whole["mask"][4:], part["mask"])
    assert np.array_equal(whole["rate"][4:], part["rate"]) and whole["drop_seed"] == p["drop_seed"]
    assert ((whole["rate"] >= 0.1) & (whole["rate"] < 0.3)).all()
    op = t.chain_op(p, torch.zeros(2, 2, 4, 4, 4))
    assert op.kind == L.BA_OP_DROPOUT and op.flags == L.BA_DROPOUT_CHANNEL
    assert op.seed == p["drop_seed"] and op.elem_offset == 4
    assert ba.NormalizeIntensityd(["x"], channel_wise=False).transform.channel_wise is False


def _calls(ops, x, w):
    return {"dropout": lambda: ops.dropout(x, 0.5, 1), "group_norm": lambda: ops.group_norm(x, 2),
            "weight": lambda: ops.group_norm(torch.zeros(2, 4, 3, 3, 3), 2, w),
            "rate": lambda: ops.dropout(torch.zeros(4, 2, 3, 3, 3), w, 1)}


@pytest.mark.parametrize("name", ["dropout", "group_norm", "weight", "rate"])
def test_forward_mode_is_refused(ba, name):
    """A tangent that the launch would drop; without one the call goes on (and
    ends at the CPU tensor)."""
    from batchaug_b200 import ops
    x, w = torch.zeros(2, 4, 3, 3, 3), torch.ones(4)
    with torch.autograd.forward_ad.dual_level():
        dual = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _calls(ops, *dual)[name]()
        with pytest.raises(ValueError, match="CUDA"):
            _calls(ops, x, w)[name]()


@pytest.mark.parametrize("name", ["dropout", "group_norm"])
def test_a_recorded_call_is_refused(ba, name):
    """Such a recording would hold the allocation and not the launch."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from batchaug_b200 import ops
    x = torch.zeros(2, 4, 3, 3, 3)

    def f(t):
        return _calls(ops, t, None)[name]()
    for record in (lambda: torch.jit.trace(f, (x,)), lambda: make_fx(f)(x),
                   lambda: make_fx(f, pre_dispatch=True)(x)):
        with pytest.raises(NotImplementedError, match="recorded"):
            record()


def test_queries_and_launches_are_made_on_the_tensors_device(ba, monkeypatch):
    """The scratch of a call is asked for where the call is made, and with the
    result's address in the descriptor (here another device than the current
    one: the CPU, the library's calls replaced by records of it)."""
    import contextlib

    from batchaug_b200 import _lib as L
    from batchaug_b200 import ops
    current, calls = [], []

    @contextlib.contextmanager
    def device(d):
        current.append(d)
        yield
        current.pop()

    class Lib:
        def __getattr__(self, name):
            def call(desc, *args):
                calls.append((name, current[-1:], getattr(desc._obj, "out", 1)))
                return 64 if name == "ba_norm_workspace_bytes" else 0
            return call
    x = torch.zeros(2, 4, 3, 3, 3, requires_grad=True)
    monkeypatch.setattr(ops, "_feature_map", lambda t, name: (t, L.BA_CHANNELS_FIRST))
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice",
                        lambda: current[-1].index if current else 0, raising=False)
    monkeypatch.setattr(L, "stream_ptr", lambda d: 0)
    monkeypatch.setattr(L, "lib", Lib())
    w = torch.ones(4, requires_grad=True)
    for y in (ops.group_norm(x, 2, w), ops.dropout(x, 0.5, 1)):
        torch.autograd.grad(y, x, torch.ones_like(x))
    assert [c[0] for c in calls] == ["ba_norm_workspace_bytes", "ba_norm_forward", "ba_dropout",
                                     "ba_norm_workspace_bytes", "ba_norm_backward", "ba_dropout"]
    assert all(c[1] == [x.device] and c[2] for c in calls), calls
    assert not current


def test_groups_too_wide_for_a_cluster_are_cut_for_the_device(ba):
    """More channels than a cluster's 64 warps: the unit is cut into as many
    parts as its channels have tiles of 256 voxels (eight tiles a part), not into
    whole channels, as the size of the scratch shows (16 bytes and 16 a part)."""
    from batchaug_b200 import _lib as L
    for channels, n, tiles in ((128, 10, 4), (72, 8, 2), (256, 6, 1)):
        d = _norm(L, batch=1, channels=channels, groups=1, H=n, W=n, D=n, dtype=L.BA_BF16,
                  layout=L.BA_CHANNELS_FIRST)
        size = L.lib.ba_norm_workspace_bytes(ctypes.byref(d), 0)
        assert size == 16 + 16 * channels * tiles // 8


def test_rows_too_long_for_a_stride_are_refused(ba):
    """Channels last, a block of columns one access wide (the number of accesses
    in a row has no small divisor): its threads are 256 rows apart, and 256 rows
    of so many channels are 2^32 bytes."""
    from batchaug_b200 import _lib as L
    prime = 1048583
    assert all(prime % k for k in range(2, 1025))
    d = _norm(L, batch=1, channels=4 * prime, groups=4 * prime, H=2, W=1, D=1,
              out=1 << 30, dy=1 << 32)
    for fn in (L.lib.ba_norm_forward, L.lib.ba_norm_backward):
        assert fn(ctypes.byref(d), 1 << 34, 1 << 40, None) == L.BA_EUNSUPPORTED
        assert b"too large" in L.lib.ba_last_error()
    # one row's bytes less
    d.channels = d.groups = 4 * 1048573
    assert L.lib.ba_norm_forward(ctypes.byref(d), None, 0, None) == L.BA_EINVAL
    assert b"workspace" in L.lib.ba_last_error()
