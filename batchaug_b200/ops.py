"""Functional entry points: torch tensors in, C-ABI calls out.

Each function validates tensors (CUDA, contiguous, fp32/bf16), allocates the
outputs and scratch with torch's caching allocator, and enqueues the kernels
on torch's current stream.  These are what the transform classes call; they
can also be used directly.
"""
from __future__ import annotations

import contextlib
import ctypes
import os

import numpy as np
import torch
from torch.autograd import forward_ad
from torch._ops import _len_torch_dispatch_stack_pre_dispatch
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib as L
from . import _timing


def _contig(t: torch.Tensor, name: str) -> torch.Tensor:
    L.require_cuda(t, name)
    return t if t.is_contiguous() else t.contiguous()


def _to_device(arr: np.ndarray, device) -> torch.Tensor:
    """Asynchronous small host-to-device copy through pinned memory."""
    t = torch.from_numpy(np.ascontiguousarray(arr))
    return t.pin_memory().to(device, non_blocking=True)


def _dev_f32(x, device, name):
    """Small parameter arrays (numpy or tensor) as contiguous fp32 on device."""
    if isinstance(x, torch.Tensor):
        return x.to(device=device, dtype=torch.float32).contiguous()
    return _to_device(np.asarray(x, dtype=np.float32), device)


def _dev_mask(mask, B, device):
    if mask is None:
        return None
    if isinstance(mask, torch.Tensor):
        m = mask.to(device=device).reshape(B)
        if m.dtype in (torch.bool, torch.uint8):
            return m.contiguous().view(torch.uint8)  # a view: no kernel
        return (m != 0).to(torch.uint8).contiguous()
    return _to_device(np.asarray(mask).reshape(B).astype(np.uint8), device)


# ---------------------------------------------------------------------------
# Geometric
# ---------------------------------------------------------------------------

# Trilinear arithmetic of the resample: False (default) interpolates with
# fused multiply-add lerps, within 1e-5 (fp32) / 2 bf16 ulp of torch's CPU
# grid_sample; True rounds every weight product and sum as torch's CPU code
# does (bit for bit).  Coordinates, and so nearest keys, are exact either way.
# BATCHAUG_B200_EXACT=1 in the environment starts in exact mode.
_EXACT = [os.environ.get("BATCHAUG_B200_EXACT", "0") == "1"]


def set_resample_exact(flag: bool) -> bool:
    """Set the default trilinear arithmetic (see above); returns the old one."""
    old, _EXACT[0] = _EXACT[0], bool(flag)
    return old


@contextlib.contextmanager
def resample_exact(flag: bool = True):
    """``with resample_exact():`` runs its body's resamples in exact mode."""
    old = set_resample_exact(flag)
    try:
        yield
    finally:
        set_resample_exact(old)


def resample3d(tensors, *, affine=None, theta=None, grid=None, modes="bilinear",
               paddings="zeros", align_corners=False, mask=None, out=None, exact=None,
               minmax=None):
    """Resample one or more (B,C,H,W,D) tensors through one shared map.

    Exactly one of ``affine`` (MONAI (B,4,4)), ``theta`` (affine_grid
    (B,3|4,4)) or ``grid`` (grid_sample (B,H,W,D,3)) gives the map.  ``modes``
    and ``paddings`` are a string or one entry per tensor.  Masked-out
    elements are copied.  ``exact`` overrides the default trilinear
    arithmetic (``set_resample_exact``).  ``minmax`` (one entry per tensor,
    None or an int32 (B, C, 2) device tensor) receives each output's
    per-(element, channel) min/max as statistics for a following
    ScaleIntensity (``ChainOp(stats=...)``).  Returns a list of new tensors
    (or fills ``out``).
    """
    single = isinstance(tensors, torch.Tensor)
    ts = [tensors] if single else list(tensors)
    if not 1 <= len(ts) <= L.BA_MAX_KEYS:
        raise ValueError(f"resample3d takes 1..{L.BA_MAX_KEYS} tensors")
    ts = [_contig(t, "tensor") for t in ts]
    for t in ts:
        if t.dim() != 5:
            raise ValueError(f"expected (B,C,H,W,D) tensors, got shape {tuple(t.shape)}")
    B, _, H, W, D = ts[0].shape
    device = ts[0].device
    for t in ts[1:]:
        if t.shape[0] != B or tuple(t.shape[2:]) != (H, W, D) or t.device != device:
            raise ValueError("resample3d: tensors must share batch, spatial shape and device")
    modes = [modes] * len(ts) if isinstance(modes, str) else list(modes)
    paddings = [paddings] * len(ts) if isinstance(paddings, str) else list(paddings)
    for m in modes:
        if m not in L.MODES:
            raise ValueError(f"unsupported interpolation mode {m!r} (bilinear or nearest)")
    for p in paddings:
        if p not in L.PADDINGS:
            raise ValueError(f"unsupported padding_mode {p!r} (zeros, border or reflection)")
    if sum(x is not None for x in (affine, theta, grid)) != 1:
        raise ValueError("resample3d needs exactly one of affine, theta or grid")
    # host (numpy) transforms and masks ride in the kernels' parameters
    # (BA_RESAMPLE_HOST_PARAMS): no upload, no device allocation
    host = not isinstance(affine if affine is not None else theta, torch.Tensor) and \
        (grid is None or isinstance(grid, torch.Tensor)) and not isinstance(mask, torch.Tensor)
    if affine is not None:
        xf = (np.ascontiguousarray(affine, np.float32).reshape(B, -1) if host
              else _dev_f32(affine, device, "affine").reshape(B, -1))
        kind, stride = L.BA_XFORM_AFFINE, xf.shape[1]
        if stride != 16:
            raise ValueError("affine must be (B,4,4)")
    elif theta is not None:
        xf = (np.ascontiguousarray(theta, np.float32).reshape(B, -1) if host
              else _dev_f32(theta, device, "theta").reshape(B, -1))
        kind, stride = L.BA_XFORM_THETA, xf.shape[1]
        if stride not in (12, 16):
            raise ValueError("theta must be (B,3,4) or (B,4,4)")
    else:
        xf = _dev_f32(grid, device, "grid")
        if tuple(xf.shape) != (B, H, W, D, 3):
            raise ValueError(f"grid must be {(B, H, W, D, 3)}, got {tuple(xf.shape)}")
        kind, stride = L.BA_XFORM_GRID, 0
    if host:
        m = None if mask is None else np.ascontiguousarray(np.asarray(mask).reshape(B) != 0,
                                                           np.uint8)
    else:
        m = _dev_mask(mask, B, device)
    outs = list(out) if out is not None else [torch.empty_like(t) for t in ts]
    d = L.ResampleDesc()
    d.batch, d.H, d.W, d.D = B, H, W, D
    d.xform_kind = kind
    d.align_corners = int(bool(align_corners))
    d.flags = L.BA_RESAMPLE_EXACT if (_EXACT[0] if exact is None else exact) else 0
    d.n_keys = len(ts)
    if host:
        d.flags |= L.BA_RESAMPLE_HOST_PARAMS
        d.xform = xf.ctypes.data if kind != L.BA_XFORM_GRID else xf.data_ptr()
        d.mask = None if m is None else m.ctypes.data
    else:
        d.xform = xf.data_ptr()
        d.mask = L.ptr(m)
    d.xform_stride = stride
    mms = list(minmax) if minmax is not None else [None] * len(ts)
    if len(mms) != len(ts):
        raise ValueError("resample3d: minmax needs one entry per tensor")
    for i, (t, o) in enumerate(zip(ts, outs)):
        k = d.keys[i]
        k.src, k.dst = t.data_ptr(), o.data_ptr()
        mm = mms[i]
        if mm is not None:
            if (mm.dtype != torch.int32 or tuple(mm.shape) != (B, t.shape[1], 2)
                    or not mm.is_contiguous() or mm.device != device):
                raise ValueError(f"resample3d: minmax[{i}] must be a contiguous int32 "
                                 f"{(B, t.shape[1], 2)} tensor on {device}")
            k.minmax = mm.data_ptr()
        k.channels = t.shape[1]
        k.dtype = L.dtype_code(t)
        k.mode = L.MODES[modes[i]]
        k.padding = L.PADDINGS[paddings[i]]
    tok = _timing.begin("ba_resample3d", sum(2 * t.numel() * t.element_size() for t in ts),
                        device)
    L.check(L.lib.ba_resample3d(ctypes.byref(d), L.stream_ptr(device)), "ba_resample3d")
    _timing.end(tok)
    return outs[0] if single else outs


# ---------------------------------------------------------------------------
# Intensity chain
# ---------------------------------------------------------------------------

class ChainOp:
    """One op of a fused intensity chain (device tensors for its params)."""

    __slots__ = ("kind", "flags", "mask", "param", "param2", "noise", "seed", "elem_offset",
                 "degree", "c0", "c1", "stats")

    def __init__(self, kind, flags=0, mask=None, param=None, param2=None, noise=None, seed=0,
                 elem_offset=0, degree=0, c0=0.0, c1=0.0, stats=None):
        self.kind, self.flags, self.mask = kind, flags, mask
        self.param, self.param2, self.noise = param, param2, noise
        self.seed, self.elem_offset, self.degree = seed, elem_offset, degree
        self.c0, self.c1 = c0, c1
        self.stats = stats  # RESCALE with BA_RESCALE_GIVEN: resample3d's minmax


def intensity_chain(x: torch.Tensor, ops, out: torch.Tensor | None = None,
                    inplace: bool = False) -> torch.Tensor:
    """Apply a list of ChainOp to x in as few HBM passes as possible."""
    x = _contig(x, "tensor")
    if x.dim() != 5:
        raise ValueError(f"expected a (B,C,H,W,D) tensor, got shape {tuple(x.shape)}")
    if not 1 <= len(ops) <= L.BA_MAX_OPS:
        raise ValueError(f"intensity_chain takes 1..{L.BA_MAX_OPS} ops")
    B, C, H, W, D = x.shape
    if out is None:
        out = x if inplace else torch.empty_like(x)
    d = L.ChainDesc()
    d.src, d.dst = x.data_ptr(), out.data_ptr()
    d.batch, d.channels, d.H, d.W, d.D = B, C, H, W, D
    d.dtype = L.dtype_code(x)
    d.n_ops = len(ops)
    keep = []
    for i, op in enumerate(ops):
        o = d.ops[i]
        o.kind, o.flags = op.kind, op.flags
        for name in ("mask", "param", "param2", "noise", "stats"):
            t = getattr(op, name)
            if t is not None:
                if t.device != x.device:
                    raise ValueError(f"op {i} {name} is on {t.device}, tensor on {x.device}")
                keep.append(t)
            setattr(o, name, L.ptr(t))
        o.seed = int(op.seed) & 0xFFFFFFFFFFFFFFFF
        o.elem_offset = int(op.elem_offset)
        o.degree = int(op.degree)
        o.c0, o.c1 = float(op.c0), float(op.c1)
    nbytes = L.lib.ba_intensity_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device) if nbytes else None
    tok = _timing.begin("ba_intensity_chain", 2 * x.numel() * x.element_size(), x.device)
    L.check(L.lib.ba_intensity_chain(ctypes.byref(d), L.ptr(ws), nbytes, L.stream_ptr(x.device)),
            "ba_intensity_chain")
    _timing.end(tok)
    return out


def minmax(x: torch.Tensor, n_groups: int):
    """Per-group (min, max) of x viewed as (n_groups, -1), fp32 tensors."""
    x = _contig(x, "tensor")
    if x.numel() % max(n_groups, 1):
        raise ValueError("minmax: numel is not a multiple of n_groups")
    stats = torch.empty(n_groups, 2, dtype=torch.float32, device=x.device)
    tok = _timing.begin("ba_minmax", x.numel() * x.element_size(), x.device)
    L.check(L.lib.ba_minmax(x.data_ptr(), L.dtype_code(x), n_groups,
                            x.numel() // max(n_groups, 1), stats.data_ptr(),
                            L.stream_ptr(x.device)), "ba_minmax")
    _timing.end(tok)
    return stats[:, 0], stats[:, 1]


# ---------------------------------------------------------------------------
# Smoothing / elastic
# ---------------------------------------------------------------------------

def gauss_taps_len(max_sigma: float, truncated: float) -> int:
    return int(L.lib.ba_gauss_taps_len(float(max_sigma), float(truncated)))


def gauss_taps(sigmas: torch.Tensor, K: int) -> torch.Tensor:
    """(B,K) taps of gaussian_1d_batch for sigmas already on device."""
    s = sigmas.to(torch.float32).contiguous()
    L.require_cuda(s, "sigmas")
    taps = torch.empty(s.numel(), K, dtype=torch.float32, device=s.device)
    L.check(L.lib.ba_gauss_taps(s.data_ptr(), s.numel(), K, taps.data_ptr(),
                                L.stream_ptr(s.device)), "ba_gauss_taps")
    return taps


def smooth3d(x: torch.Tensor, taps_h, taps_w, taps_d, mask=None,
             padding_mode=None) -> torch.Tensor:
    """Separable Gaussian smoothing with per-element taps; padding_mode is
    None/"constant" (zeros), "reflect" or "replicate" as in F.pad."""
    if padding_mode not in L.SMOOTH_PADS:
        raise ValueError(f"unsupported padding_mode {padding_mode!r}")
    x = _contig(x, "tensor")
    B, C, H, W, D = x.shape
    th, tw, td = (_dev_f32(t, x.device, "taps") for t in (taps_h, taps_w, taps_d))
    m = _dev_mask(mask, B, x.device)
    out = torch.empty_like(x)
    nbytes = L.lib.ba_smooth_workspace_bytes(B, C, H, W, D)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    tok = _timing.begin("ba_smooth3d", 2 * x.numel() * x.element_size(), x.device)
    L.check(L.lib.ba_smooth3d(x.data_ptr(), out.data_ptr(), L.dtype_code(x), B, C, H, W, D,
                              th.data_ptr(), th.shape[1], tw.data_ptr(), tw.shape[1],
                              td.data_ptr(), td.shape[1], L.SMOOTH_PADS[padding_mode], L.ptr(m),
                              ws.data_ptr(), nbytes,
                              L.stream_ptr(x.device)), "ba_smooth3d")
    _timing.end(tok)
    return out


def sharpen3d(x: torch.Tensor, taps1, taps2, alpha, mask=None,
              padding_mode=None) -> torch.Tensor:
    """Unsharp masking blurred + alpha * (blurred - double_blurred) with
    per-element taps: taps1 / taps2 are (H, W, D) triples of (B, K) for the
    first and second blur."""
    if padding_mode not in L.SMOOTH_PADS:
        raise ValueError(f"unsupported padding_mode {padding_mode!r}")
    x = _contig(x, "tensor")
    B, C, H, W, D = x.shape
    t1 = [_dev_f32(t, x.device, "taps1") for t in taps1]
    t2 = [_dev_f32(t, x.device, "taps2") for t in taps2]
    for t in t1 + t2:
        if t.dim() != 2 or t.shape[0] != B:
            raise ValueError(f"taps must be (B={B}, K), got {tuple(t.shape)}")
    al = _dev_f32(alpha, x.device, "alpha").reshape(-1)
    if al.numel() != B:
        raise ValueError(f"alpha has {al.numel()} values for a batch of {B}")
    m = _dev_mask(mask, B, x.device)
    out = torch.empty_like(x)
    d = L.SharpenDesc()
    d.src, d.dst = x.data_ptr(), out.data_ptr()
    d.dtype, d.padding = L.dtype_code(x), L.SMOOTH_PADS[padding_mode]
    d.batch, d.channels, d.H, d.W, d.D = B, C, H, W, D
    for i in range(3):
        d.taps1[i], d.K1[i] = t1[i].data_ptr(), t1[i].shape[1]
        d.taps2[i], d.K2[i] = t2[i].data_ptr(), t2[i].shape[1]
    d.alpha, d.mask = al.data_ptr(), L.ptr(m)
    nbytes = L.lib.ba_sharpen_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    tok = _timing.begin("ba_sharpen3d", 2 * x.numel() * x.element_size(), x.device)
    L.check(L.lib.ba_sharpen3d(ctypes.byref(d), ws.data_ptr(), nbytes, L.stream_ptr(x.device)),
            "ba_sharpen3d")
    _timing.end(tok)
    return out


def lowres3d(x: torch.Tensor, zoom, mask=None, downsample_mode="nearest",
             upsample_mode="trilinear", align_corners=False, max_zoom=None) -> torch.Tensor:
    """Down to max(1, rint(s * zoom[b])) per axis and back up, per element
    (RandSimulateLowResolution.apply).  max_zoom bounds zoom (read from it
    when None, which costs a device-to-host copy for a device tensor)."""
    for m in (downsample_mode, upsample_mode):
        if m not in L.INTERP_MODES:
            raise ValueError(f"unsupported interpolation mode {m!r} for a 5-D tensor "
                             f"(expected one of {sorted(L.INTERP_MODES)})")
    x = _contig(x, "tensor")
    B, C, H, W, D = x.shape
    z = _dev_f32(zoom, x.device, "zoom").reshape(-1)
    if z.numel() != B:
        raise ValueError(f"zoom has {z.numel()} values for a batch of {B}")
    if max_zoom is None:
        max_zoom = float(z.max()) if B else 1.0
    m = _dev_mask(mask, B, x.device)
    out = torch.empty_like(x)
    d = L.LowresDesc()
    d.src, d.dst, d.dtype = x.data_ptr(), out.data_ptr(), L.dtype_code(x)
    d.down_mode, d.up_mode = L.INTERP_MODES[downsample_mode], L.INTERP_MODES[upsample_mode]
    d.align_corners = int(bool(align_corners))
    d.batch, d.channels, d.H, d.W, d.D = B, C, H, W, D
    d.zoom, d.mask, d.max_zoom = z.data_ptr(), L.ptr(m), float(max(max_zoom, 1e-30))
    nbytes = L.lib.ba_lowres_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    tok = _timing.begin("ba_lowres3d", 2 * x.numel() * x.element_size(), x.device)
    L.check(L.lib.ba_lowres3d(ctypes.byref(d), ws.data_ptr(), nbytes, L.stream_ptr(x.device)),
            "ba_lowres3d")
    _timing.end(tok)
    return out


def compose_field(field: torch.Tensor, theta, mask_field=None, mask_affine=None) -> torch.Tensor:
    """Grid (B,H,W,D,3) of the elastic field ``field`` followed by the affine
    ``theta`` (B,3,4) (see ba_compose_field): one grid_sample with it
    (align_corners=True) gives I(field(A(p)))."""
    field = _contig(field.to(torch.float32), "field")
    if field.dim() != 5 or field.shape[-1] != 3:
        raise ValueError(f"field must be (B,H,W,D,3), got {tuple(field.shape)}")
    B, H, W, D, _ = field.shape
    th = _dev_f32(theta, field.device, "theta").reshape(B, -1)
    if th.shape[1] == 16:
        th = th.reshape(B, 4, 4)[:, :3, :].contiguous()
    th = th.reshape(B, 3, 4).contiguous()
    mf = _dev_mask(mask_field, B, field.device)
    ma = _dev_mask(mask_affine, B, field.device)
    out = torch.empty_like(field)
    tok = _timing.begin("ba_compose_field", 2 * field.numel() * 4, field.device)
    L.check(L.lib.ba_compose_field(field.data_ptr(), th.data_ptr(), L.ptr(mf), L.ptr(ma), B, H, W,
                                   D, out.data_ptr(), L.stream_ptr(field.device)),
            "ba_compose_field")
    _timing.end(tok)
    return out


def elastic_grid(shape, taps, magnitude, *, u=None, seed=0, elem_offset=0,
                 device=None) -> torch.Tensor:
    """grid_sample grid (B,H,W,D,3) of Rand3DElastic from taps (B,K) and
    magnitude (B,); the uniform draw u (B,3,H,W,D) is generated in-kernel
    from (seed, elem_offset) unless given."""
    B, H, W, D = shape
    device = device or (u.device if u is not None else taps.device)
    tp = _dev_f32(taps, device, "taps")
    mg = _dev_f32(magnitude, device, "magnitude").reshape(B)
    uu = None if u is None else _contig(u.to(torch.float32), "u")
    grid = torch.empty(B, H, W, D, 3, dtype=torch.float32, device=device)
    nbytes = L.lib.ba_elastic_workspace_bytes(B, H, W, D)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
    tok = _timing.begin("ba_elastic_grid", grid.numel() * 4, device)
    L.check(L.lib.ba_elastic_grid(L.ptr(uu), int(seed) & 0xFFFFFFFFFFFFFFFF, int(elem_offset),
                                  B, H, W, D, tp.data_ptr(), tp.shape[1], mg.data_ptr(),
                                  grid.data_ptr(), ws.data_ptr(), nbytes,
                                  L.stream_ptr(device)), "ba_elastic_grid")
    _timing.end(tok)
    return grid


# ---------------------------------------------------------------------------
# Feature maps: dropout and group norm (differentiable)
# ---------------------------------------------------------------------------

# What _refuse_unseen looks into, and an ordinary call has none of: asked for in
# line, 0.3 us of a call of 8
_is_tracing, _modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
_modes_before_autograd = _len_torch_dispatch_stack_pre_dispatch


def _refuse_unseen(name: str, *args) -> None:
    """Refuses a call that something watches which cannot see the launch behind
    it: forward-mode differentiation would take the result for a constant, and
    a recorded program (torch.jit.trace, make_fx) would return memory that
    nobody wrote.  (functorch's transforms end at the tensors' addresses.)"""
    if _is_tracing() or get_proxy_mode() is not None:
        raise NotImplementedError(f"{name} cannot be recorded by torch.jit.trace or make_fx")
    if forward_ad._current_level >= 0:  # within dual_level()
        for t in args:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} has no forward-mode derivative")


def _feature_map(x: torch.Tensor, name: str):
    """``x`` dense in one of the two layouts the kernels take, and which: a
    (B,C,H,W,D) tensor contiguous as named or in torch.channels_last_3d is
    taken as it is, any other strides are copied to the former."""
    if not x.is_cuda:
        L.require_cuda(x, name)
    if x.dim() != 5:
        raise ValueError(f"expected a (B,C,H,W,D) tensor, got shape {tuple(x.shape)}")
    if x.is_contiguous(memory_format=torch.channels_last_3d):
        # one channel or one voxel: both layouts at once, and what is contiguous
        # is the longer axis
        return x, (L.BA_CHANNELS_FIRST if x.shape[1] == 1 else L.BA_CHANNELS_LAST)
    return (x if x.is_contiguous() else x.contiguous()), L.BA_CHANNELS_FIRST


def _like(t: torch.Tensor, x: torch.Tensor, layout: int) -> torch.Tensor:
    """``t`` (a gradient) with x's dtype and layout."""
    if t.dtype is not x.dtype:
        t = t.to(x.dtype)
    f = (torch.channels_last_3d if layout == L.BA_CHANNELS_LAST else torch.contiguous_format)
    return t if t.is_contiguous(memory_format=f) else t.contiguous(memory_format=f)


def _drop_params(x: torch.Tensor, p, seed, name: str):
    """Checked (p, p_elem, seed, seed_dev): a probability in [0, 1] or a (B,)
    tensor of them, and an integer seed or an int64 CUDA tensor holding one."""
    p_elem = seed_dev = None
    if isinstance(p, torch.Tensor):
        if p.numel() != x.shape[0]:
            raise ValueError(f"{name}: p has {p.numel()} values for a batch of {x.shape[0]}")
        p_elem = p.detach().to(device=x.device, dtype=torch.float32).reshape(-1).contiguous()
        p = 0.0
    elif not 0.0 <= p <= 1.0:
        raise ValueError(f"{name}: p={p} is not a probability")
    if seed is None:
        if p_elem is not None or p > 0.0:
            raise ValueError(f"{name}: dropout needs a seed")
        seed = 0
    elif isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError(f"{name}: a seed tensor must be one int64 on {x.device}")
        seed_dev, seed = seed, 0
    return p, p_elem, int(seed) & 0xFFFFFFFFFFFFFFFF, seed_dev


def _launch(fn, name: str, passes: int, x: torch.Tensor, *args) -> None:
    """One C entry on the current stream of x's device, which is current (it
    answers for the query of a call's scratch too); ``passes``: how often it
    moves x's bytes."""
    device = x.device
    if _timing._active is None:
        st = fn(*args, L.stream_ptr(device))
    else:
        tok = _timing.begin(name, passes * x.numel() * x.element_size(), device)
        st = fn(*args, L.stream_ptr(device))
        _timing.end(tok)
    if st:
        L.check(st, name)


def _once_differentiable(backward):
    """torch's once_differentiable, whose wrapper costs a small backward pass
    3 us, where it is not idle: while the pass itself is being recorded."""
    recorded = torch.autograd.function.once_differentiable(backward)

    def call(ctx, dy):
        return (recorded if torch.is_grad_enabled() else backward)(ctx, dy)
    return call


def _dropout_call(x, desc):
    if x.device.index != torch._C._cuda_getDevice():  # current_device() without its checks
        with torch.cuda.device(x.device):
            return _dropout_call(x, desc)
    out = torch.empty_like(x)
    desc.src, desc.dst = x.data_ptr(), out.data_ptr()
    _launch(L.lib.ba_dropout, "ba_dropout", 2, x, ctypes.byref(desc))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, call):
        desc, _, tensors = ctx.call = call
        # the tensors behind the descriptor's addresses, if it has any
        if tensors:
            ctx.save_for_backward(*tensors)
        return _dropout_call(x, desc)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        desc, layout, tensors = ctx.call
        if _is_tracing() or _modes() or _modes_before_autograd() or forward_ad._current_level >= 0:
            _refuse_unseen("dropout", dy)
        if tensors:
            ctx.saved_tensors  # raises if one of them was written to since
        # the same draw on the gradient
        return _dropout_call(_like(dy, dy, layout), L.DropoutDesc.from_buffer_copy(desc)), None


def dropout(x: torch.Tensor, p, seed, *, mask=None, elem_offset: int = 0,
            channelwise: bool = False, rescale: bool = True) -> torch.Tensor:
    """Zero each voxel of x (B,C,H,W,D) with probability ``p`` and scale the
    others by 1 / (1 - p) (``rescale``); ``channelwise`` draws once for each
    (element, channel).  Differentiable (once, in reverse mode; forward mode and
    a recorded call are refused); the mask is never stored, the backward pass
    draws it again.

    ``p``: a number, or a (B,) tensor with a rate for each element.  ``mask``
    (B,): elements left as they are where false.  ``seed``: an integer, or a
    CUDA int64 tensor of one value that the kernel reads when it runs, so a
    captured graph draws other bits after the caller has changed it (the
    backward pass must see the value that the forward pass saw).  The bits
    depend on (seed, elem_offset + element, channel, voxel) only, not on
    the memory layout, which the result shares with x."""
    if _is_tracing() or _modes() or _modes_before_autograd() or forward_ad._current_level >= 0:
        _refuse_unseen("dropout", x, p)
    x, layout = _feature_map(x, "x")
    dtype = L.dtype_code(x)
    p, p_elem, seed, seed_dev = _drop_params(x, p, seed, "dropout")
    m = _dev_mask(mask, x.shape[0], x.device)
    flags = (L.BA_DROPOUT_CHANNEL if channelwise else 0) | (L.BA_DROPOUT_RESCALE if rescale else 0)
    B, C, H, W, D = x.shape
    desc = L.dropout_desc(0, 0, B, C, H, W, D, dtype, layout, flags, p,
                          0 if p_elem is None else p_elem.data_ptr(),
                          0 if m is None else m.data_ptr(), seed,
                          0 if seed_dev is None else seed_dev.data_ptr(),
                          int(elem_offset) & 0xFFFFFFFFFFFFFFFF)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, (desc, layout,
                                  [t for t in (p_elem, m, seed_dev) if t is not None]))
    return _dropout_call(x, desc)


def _norm_forward(x, desc, groups):
    """y, and the buffer of the statistics (and, behind them, the scratch)."""
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return _norm_forward(x, desc, groups)
    y = torch.empty_like(x)
    desc.out = y.data_ptr()
    size = L.lib.ba_norm_workspace_bytes(ctypes.byref(desc), 0)
    head = (x.shape[0] * groups * 8 + 15) & ~15
    buf = torch.empty(head + size, dtype=torch.uint8, device=x.device)
    at = buf.data_ptr()
    desc.stats = at
    _launch(L.lib.ba_norm_forward, "ba_norm_forward", 2, x, ctypes.byref(desc), at + head, size)
    return y, buf


def _norm_backward(x, desc):
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return _norm_backward(x, desc)
    size = L.lib.ba_norm_workspace_bytes(ctypes.byref(desc), 1)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    _launch(L.lib.ba_norm_backward, "ba_norm_backward", 3, x, ctypes.byref(desc), ws.data_ptr(),
            size)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, call):
        desc, groups, _, tensors = ctx.call = call
        y, buf = _norm_forward(x, desc, groups)
        # x, the parameters, and what else the descriptor points to
        ctx.save_for_backward(x, weight, bias, buf, *tensors)
        return y

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        if _is_tracing() or _modes() or _modes_before_autograd() or forward_ad._current_level >= 0:
            _refuse_unseen("group_norm", dy)
        x, weight, bias, buf = ctx.saved_tensors[:4]
        desc, _, layout, _ = ctx.call
        desc = L.NormDesc.from_buffer_copy(desc)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        # what hooks on saved tensors give back (offloading, recomputation)
        # lies elsewhere, and may have lost its strides
        x = _like(x, x, layout)
        desc.x, desc.stats = x.data_ptr(), buf.data_ptr()
        desc.weight = None if weight is None else weight.data_ptr()
        desc.bias = None if bias is None else bias.data_ptr()
        dy = _like(dy, x, layout)
        dx = dw = db = None
        desc.dy, desc.out = dy.data_ptr(), None
        if need_x:
            dx = torch.empty_like(x)
            desc.out = dx.data_ptr()
        if need_w:
            dw = torch.empty_like(weight)
            desc.dweight = dw.data_ptr()
        if need_b:
            db = torch.empty_like(bias)
            desc.dbias = db.data_ptr()
        _norm_backward(x, desc)
        return dx, dw, db, None


def _norm_param(t, x, name):
    if t.device != x.device:
        raise ValueError(f"group_norm: {name} is on {t.device}, x on {x.device}")
    if t.dim() != 1 or t.shape[0] != x.shape[1]:
        raise ValueError(f"group_norm: {name} must be ({x.shape[1]},), got {tuple(t.shape)}")
    L.dtype_code(t)
    return t if t.is_contiguous() else t.contiguous()


def group_norm(x: torch.Tensor, num_groups: int, weight=None, bias=None, *, eps: float = 1e-5,
               activation=None, negative_slope: float = 0.01, p=0.0, seed=None,
               elem_offset: int = 0) -> torch.Tensor:
    """dropout(activation(group_norm(x) * weight + bias)) of x (B,C,H,W,D),
    each group of C / num_groups consecutive channels of an element
    normalised by its own mean and biased variance.  Differentiable in x,
    weight and bias (once, in reverse mode; forward mode and a recorded call
    are refused).

    ``activation``: None (or "none"), "relu", "leaky_relu" (with
    ``negative_slope``), "silu" or "gelu" (exact).  ``weight`` and ``bias``
    (C,), float32 or bfloat16 (the same for both), or None.  ``p``, ``seed``
    and ``elem_offset``: as in :func:`dropout`, rescaled; no dropout by
    default.  x may be contiguous or in torch.channels_last_3d, and the
    result is laid out as it is."""
    if _is_tracing() or _modes() or _modes_before_autograd() or forward_ad._current_level >= 0:
        _refuse_unseen("group_norm", x, weight, bias, p)
    x, layout = _feature_map(x, "x")
    dtype = L.dtype_code(x)
    num_groups = int(num_groups)
    if num_groups < 1 or x.shape[1] % num_groups:
        raise ValueError(f"group_norm: {num_groups} groups do not divide {x.shape[1]} channels")
    if activation not in L.ACTIVATIONS:
        raise ValueError(f"unsupported activation {activation!r} (expected one of "
                         f"{[a for a in L.ACTIVATIONS if a]})")
    param = None
    if weight is not None:
        param = weight = _norm_param(weight, x, "weight")
    if bias is not None:
        bias = _norm_param(bias, x, "bias")
        if param is None:
            param = bias
        elif param.dtype is not bias.dtype:
            raise ValueError(f"group_norm: weight is {weight.dtype}, bias {bias.dtype}")
    p, p_elem, seed, seed_dev = _drop_params(x, p, seed, "group_norm")
    B, C, H, W, D = x.shape
    desc = L.norm_desc(x.data_ptr(), 0, 0, 0 if weight is None else weight.data_ptr(),
                       0 if bias is None else bias.data_ptr(), 0, 0, 0, B, C, H, W, D, num_groups,
                       dtype, layout, L.BA_F32 if param is None else L.dtype_code(param),
                       L.ACTIVATIONS[activation], eps, negative_slope, p, 0,
                       0 if p_elem is None else p_elem.data_ptr(), seed,
                       0 if seed_dev is None else seed_dev.data_ptr(),
                       int(elem_offset) & 0xFFFFFFFFFFFFFFFF)
    if (x.requires_grad or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)) and torch.is_grad_enabled():
        tensors = [t for t in (p_elem, seed_dev) if t is not None]
        return _GroupNorm.apply(x, weight, bias, (desc, num_groups, layout, tensors))
    return _norm_forward(x, desc, num_groups)[0]


def host_rand_affine(u, prob, a, b, c, present, groups, spatial_shape, mask, affine, theta):
    """ba_host_rand_affine into the given numpy outputs (mask u8 (B,),
    affine and theta (B,4,4) float32)."""
    H, W, D = spatial_shape
    B = u.shape[0]
    L.lib.ba_host_rand_affine(u.ctypes.data, B, u.shape[1], float(prob), a.ctypes.data,
                              b.ctypes.data, c.ctypes.data, int(present), int(groups), H, W, D,
                              mask.ctypes.data, affine.ctypes.data, theta.ctypes.data)


def host_uniform(seed: int, stream: int, elem_offset: int, n_elems: int,
                 per_elem: int) -> np.ndarray:
    """(n_elems, per_elem) uniforms in [0,1) keyed on global element index."""
    out = np.empty((n_elems, per_elem), np.float32)
    if n_elems and per_elem:
        L.lib.ba_host_uniform(int(seed) & 0xFFFFFFFFFFFFFFFF, int(stream) & 0xFFFF,
                              int(elem_offset), n_elems, per_elem, out.ctypes.data)
    return out

