"""RandVoxelDropout and NormalizeIntensity in the framework's own paths: alone,
as ops of a fused intensity chain, in a lazy Compose, sharded, and in front of
a training step of a network's first block.

Dropout keeps or drops exactly as the definition says and multiplies once in
the tensor's type, so chains are compared bit for bit with the ops one by one."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import feature_ref as R

pytestmark = pytest.mark.gpu


def _vol(shape, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(*shape, generator=g) + 0.25).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(5, 3, 8, 6, 4), (4, 2, 5, 7, 3), (3, 9, 4, 4, 2)])
@pytest.mark.parametrize("channel_wise", [False, True])
@pytest.mark.parametrize("rescale", [False, True])
def test_transform_is_the_operator(ba, shape, dtype, channel_wise, rescale):
    x = _vol(shape, dtype)
    t = ba.RandVoxelDropout(prob=0.7, rate=(0.1, 0.6), channel_wise=channel_wise, rescale=rescale)
    torch.manual_seed(3)
    p = t.sample_params(shape[0], shape, x.device)
    assert 0 < p["_host"]["mask"].sum() < shape[0]
    y = t.apply(x, p)
    f = R.factor(shape, p["_host"]["rate"], p["drop_seed"], channelwise=channel_wise,
                 rescale=rescale, mask=p["_host"]["mask"])
    assert torch.equal(y.cpu() != 0, f != 0)
    want = ba.dropout(x, p["rate"], p["drop_seed"], mask=p["mask"], channelwise=channel_wise,
                      rescale=rescale)
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(4, 2, 8, 8, 8), (3, 2, 5, 5, 3)])
def test_chain_is_its_ops_one_by_one(ba, shape, dtype):
    """Noise, dropout, scale, dropout, min/max rescale fused, and apart."""
    x = _vol(shape, dtype)
    ts = [ba.RandGaussianNoise(prob=0.8, std=0.2), ba.RandVoxelDropout(prob=0.8, rate=0.25),
          ba.RandScaleIntensity(prob=1.0, factors=(0.1, 0.4)),
          ba.RandVoxelDropout(prob=0.8, rate=(0.0, 0.5), rescale=True),
          ba.ScaleIntensity()]
    torch.manual_seed(7)
    params = [t.sample_params(shape[0], shape, x.device) for t in ts]
    fused = ba.ops.intensity_chain(x, [t.chain_op(p, x) for t, p in zip(ts, params)])
    y = x
    for t, p in zip(ts, params):
        y = t.apply(y, p)
    assert torch.equal(fused, y)


def test_compose_and_shards(ba):
    """A lazy Compose with both transforms; two half batches give the whole's
    elements, and every key of a dict gets the same mask."""
    B, shape = 4, (4, 2, 16, 12, 8)
    data = {"vol": _vol(shape), "aux": _vol((B, 1, 16, 12, 8), seed=1)}

    def pipeline():
        return ba.Compose([
            ba.RandAxisFlipd(["vol", "aux"], prob=0.5),
            ba.RandAffined(["vol", "aux"], prob=0.7, rotate_range=0.3),
            ba.RandGaussianNoised(["vol"], prob=1.0, std=0.05),
            ba.RandVoxelDropoutd(["vol", "aux"], prob=0.9, rate=(0.2, 0.5)),
            ba.NormalizeIntensityd(["vol"]),
        ], lazy=True)

    torch.manual_seed(11)
    whole = pipeline()(data)
    halves = []
    for off in (0, 2):
        torch.manual_seed(11)
        with ba.shard(off, B):
            halves.append(pipeline()({k: v[off:off + 2] for k, v in data.items()}))
    for k in data:
        assert torch.equal(whole[k], torch.cat([h[k] for h in halves]))
    v = whole["vol"].double()
    # fp32 z-scores: mean and variance of n = 1536 values within n half steps
    assert v.mean((2, 3, 4)).abs().max() <= 1536 * 2.0**-24
    assert (v.var((2, 3, 4), correction=0) - 1).abs().max() <= 1e-3  # eps 1e-5 of a variance >= 0.01
    # the same draws for every key: a channel has the same mask in each
    ones = ba.RandVoxelDropoutd(["a", "b"], prob=0.7, rate=0.5)(
        {"a": torch.ones(shape, device="cuda"), "b": torch.ones(4, 1, 16, 12, 8, device="cuda")})
    assert torch.equal(ones["a"][:, :1], ones["b"]) and bool((ones["b"] == 0).any())


def test_normalize_intensity(ba):
    shape = (2, 3, 9, 8, 7)
    for dtype in (torch.float32, torch.bfloat16):
        x = _vol(shape, dtype)
        for cw, groups in ((True, 3), (False, 1)):
            y = ba.NormalizeIntensity(channel_wise=cw)(x)
            ref, _ = R.norm(x.double().cpu(), groups)
            # values of order 1 about a mean of half the spread: 2^-19 (a few
            # hundred half steps) of fp32 arithmetic, half a step of the store
            tol = 2.0**-15 + torch.finfo(dtype).eps / 2 * ref.abs()
            assert ((y.double().cpu() - ref).abs() <= tol).all()
    x = _vol(shape).requires_grad_()
    (dx,) = torch.autograd.grad(ba.NormalizeIntensity()(x).square().sum(), x)
    assert torch.isfinite(dx).all()


def test_rates_out_of_range(ba):
    for bad in (-0.1, 1.5, (0.5, 0.2), (0.5, 1.1)):
        with pytest.raises(ValueError, match="rate"):
            ba.RandVoxelDropout(rate=bad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_first_block_of_a_network(ba, dtype):
    """An augmented batch, made channels last, through a pointwise product,
    normalised, activated and dropped, with all gradients: against the
    definition in 64 bits on the same intermediate."""
    shape, width = (2, 4, 10, 9, 8), 24
    torch.manual_seed(5)
    pipe = ba.Compose([ba.RandAxisFlipd(["x"], prob=0.5), ba.RandVoxelDropoutd(["x"], prob=1.0),
                       ba.NormalizeIntensityd(["x"])], lazy=True)
    x = pipe({"x": _vol(shape, dtype)})["x"]
    g = torch.Generator().manual_seed(9)
    mix = (torch.randn(width, shape[1], generator=g) / 2).to(dtype).cuda()
    h = torch.einsum("bchwd,ec->behwd", x, mix).contiguous(memory_format=torch.channels_last_3d)
    h.requires_grad_()
    w = (1 + 0.1 * torch.randn(width, generator=g)).cuda().requires_grad_()
    b = (0.1 * torch.randn(width, generator=g)).cuda().requires_grad_()
    y = ba.group_norm(h, 6, w, b, activation="gelu", p=0.15, seed=21)
    dy = torch.randn(*y.shape, generator=g).to(dtype)
    grads = torch.autograd.grad(y, [h, w, b], dy.cuda())
    l64 = [t.detach().double().cpu().contiguous().requires_grad_() for t in (h, w, b)]
    ref, _ = R.norm(l64[0], 6, l64[1], l64[2], act="gelu", f=R.factor(tuple(y.shape), 0.15, 21))
    refs = torch.autograd.grad(ref, l64, dy.double())
    # 2^-15 of values of order one is several hundred fp32 half steps
    for got, want in [(y, ref.detach()), (grads[0], refs[0])]:
        tol = 2.0**-15 * (1 + want.abs().max()) + torch.finfo(dtype).eps / 2 * want.abs()
        assert ((got.detach().double().cpu() - want).abs() <= tol).all()
    for got, want in zip(grads[1:], refs[1:]):
        # sums over 1440 terms of order one, each within 2^-17 or so
        assert ((got.double().cpu() - want).abs() <= 1440 * 2.0**-17).all()
