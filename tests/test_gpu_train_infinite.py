"""Infinities in the operands of the training operators: a result is infinite or
NaN where its definition in 64 bits is, and finite where that is.  Tolerances of
the finite ones count roundings of U = 2^-24 as for finite operands: 34 of the
sum S of a dot's magnitudes in z (none of an infinite z), 16 in a row's gradient
besides, and one a row in a sum."""
import math

import pytest
import torch

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


def _same(got, want, tol, what):
    got = got.double().cpu().reshape(want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    far = torch.isinf(want)
    assert torch.equal(got[far], want[far]) and not torch.isinf(got[~far]).any(), what
    near = torch.isfinite(want)
    assert bool(((got - want).abs() <= tol)[near].all()), what


def _sums(x, g, eg):
    """sum_r g x and sum_r g of [m, r, 32] and [m, r, h], with tolerances."""
    r = x.shape[1]
    p = g[:, :, :, None] * x[:, :, None]          # [m, r, h, 32] (0 * inf: NaN, as it is defined)
    ep = eg[:, :, :, None] * x.abs()[:, :, None]
    ep = torch.where(torch.isfinite(ep), ep, torch.zeros_like(ep))
    size = torch.where(torch.isfinite(p), p.abs(), torch.zeros_like(p))
    return (p.sum(1), ep.sum(1) + (r + 2) * U * size.sum(1) + 1e-40,
            g.sum(1), eg.sum(1) + (r + 2) * U * g.abs().sum(1) + 1e-40)


def _few_bits(shape, g, scale):
    """Values of which `scale` times each, rounded, has 8 bits."""
    v = (1.0 + torch.arange(128) / 128.0).to(torch.float32)  # every bfloat16 in [1, 2)
    k = torch.float32
    near = (v.double() / scale).to(k)
    for step in range(-2, 3):  # the nearby float32 whose product rounds to it, where there is one
        w = (near.view(torch.int32) + step).view(k)
        hit = (w * torch.tensor(scale, dtype=k)) == v
        near = torch.where(hit, w, near)
    near = near[(near * torch.tensor(scale, dtype=k)) == v]
    assert len(near) >= 64
    sign = torch.where(torch.rand(shape, generator=g) < 0.5, -1.0, 1.0)
    return near[torch.randint(0, len(near), shape, generator=g)] * sign


@pytest.mark.parametrize("scale", [1.0, 1.4426950408889634])
@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h", [1, 3, 6, 8, 9, 16, 20])
def test_infinite_samples(tr, h, dtype, whole, scale):
    """Infinite samples under weights of few bits, or whose products with log2 e
    are of few bits: their row's z is infinite, its slope 0, and only their own
    place's dw is NaN; for a target on the other side dw is infinite."""
    m, r = 5, 83
    g = torch.Generator().manual_seed(h)
    x = (0.25 + torch.rand(r, m, 32, generator=g)).to(DT[dtype])
    x[7, 1, 5], x[40, 2, 31], x[41, 2, 0] = math.inf, -math.inf, math.inf
    x[64, 3, 8], x[80, 4, 17] = math.inf, math.inf
    w = _few_bits((m, h, 32), g, scale)
    b = torch.randn(m, h, generator=g)
    t = (torch.rand(r, generator=g) < 0.5).float()
    c = torch.where(torch.rand(r, generator=g) < 0.5, 1.0, 0.1 + torch.rand(r, generator=g))
    dy = torch.randn(r, m, h, generator=g)
    rows = None if whole else torch.randperm(r, generator=g).to(torch.int32)
    order = torch.arange(r) if whole else rows.long()
    xd, wd = x.double()[order].transpose(0, 1), w.double()  # [m, r, 32]
    z = (xd[:, :, None] * wd[:, None]).sum(3) + b.double()[:, None]  # [m, r, h]
    size = (xd[:, :, None] * wd[:, None]).abs().sum(3) + b.double().abs()[:, None]
    dz = torch.where(torch.isinf(z), torch.zeros_like(z), 34 * U * size + 4 * U * z.abs())
    s, s1 = torch.sigmoid(z), torch.sigmoid(-z)
    dev = lambda v: None if v is None else v.cuda()

    y = tr.response(dev(x), dev(w), dev(b), rows=dev(rows))
    _same(y.permute(1, 0, 2), s, 0.25 * dz + 8 * U * s, "response")
    gr = dy.double().permute(1, 0, 2) * s * s1
    want = _sums(xd, gr, gr.abs() * (dz + 12 * U))
    dw, db, _ = tr.response_grad(dev(x), dev(w), dev(dy), dev(b), rows=dev(rows))
    _same(dw, want[0], want[1], "dw of the responses")
    _same(db, want[2], want[3], "db of the responses")
    tt, cc = t.double()[order][None, :, None], c.double()[order][None, :, None]
    gl = cc * ((1 - tt) * s - tt * s1)
    want = _sums(xd, gl, cc * ((1 - tt) * s + tt * s1) * (dz + 16 * U))
    loss, dw, db = tr.loss(dev(x), dev(w), dev(t), dev(b), weight=dev(c), rows=dev(rows))
    _same(dw, want[0], want[1], "dw of the loss")
    _same(db, want[2], want[3], "db of the loss")
    # from the side where nothing cancels: an infinite z is a loss of infinity for the target on the other
    # side, and 0 * inf for its own
    sp = torch.nn.functional.softplus
    term = cc * (tt * sp(-z) + (1 - tt) * sp(z))
    _same(loss, term.sum(1), (cc * (dz + 4 * U) + (16 + r) * U * term.abs()).sum(1), "loss")
