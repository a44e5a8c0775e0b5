"""Gradients so small that they leave float32's normal range (2^-126), by small
sample weights or small dy: they are rounded to float32's own steps of 2^-149
there, and not before.  Tolerances: U = 2^-24 as for other gradients (34 of the sum
S of a dot's magnitudes and 4 |z| in z, 16 a row, one a row in a sum), and half a
step of 2^-149 for each of a row's 6 roundings and each step of a sum."""
import pytest
import torch

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu
U, STEP = 2.0 ** -24, 2.0 ** -149
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h", [1, 4, 7, 8, 12, 16])
@pytest.mark.parametrize("size", [1e-28, 1e-31, 1e-34, 1.3e-36, 3e-38, 1e-40, 1e-43])
def test_small_gradients(tr, size, h, dtype):
    n, p = 333, 5
    g = torch.Generator().manual_seed(h)
    x = torch.rand(n, p, 32, generator=g).to(DT[dtype])
    w, b = torch.randn(p, h, 32, generator=g), torch.randn(p, h, generator=g)
    t = (torch.rand(n, generator=g) < 0.5).float()
    c = (0.5 + torch.rand(n, generator=g)) * size
    dy = torch.randn(n, p, h, generator=g) * size
    rows = torch.randint(-1, n, (n,), generator=g, dtype=torch.int32)
    ok = (rows >= 0)[:, None, None]
    at = rows.clamp_min(0).long()
    xd = x.double()[at]
    z = torch.matmul(xd.transpose(0, 1), w.double().transpose(1, 2)).transpose(0, 1) + b.double()
    dz = 34 * U * (torch.matmul(xd.transpose(0, 1), w.double().abs().transpose(1, 2)).transpose(0, 1) + b.double().abs()) \
        + 4 * U * z.abs()
    s, s1 = torch.sigmoid(z), torch.sigmoid(-z)
    tt, cc = t.double()[at][:, None, None], c.double()[at][:, None, None]

    def check(dw, db, gr, eg, what):
        gr, eg = torch.where(ok, gr, 0.0), torch.where(ok, eg, 0.0) + 3 * STEP
        want = torch.matmul(gr.permute(1, 2, 0), xd.transpose(0, 1))
        tol = torch.matmul(eg.permute(1, 2, 0), xd.transpose(0, 1)) + n * STEP \
            + (n + 2) * U * torch.matmul(gr.abs().permute(1, 2, 0), xd.transpose(0, 1))
        assert bool(((dw.double().cpu() - want).abs() <= tol).all()), what
        tol = eg.sum(0) + n * STEP + (n + 2) * U * gr.abs().sum(0)
        assert bool(((db.double().cpu() - gr.sum(0)).abs() <= tol).all()), what

    dev = [v.cuda() for v in (x, w, t, b, c, rows)]
    loss, dw, db = tr.loss(dev[0], dev[1], dev[2], dev[3], weight=dev[4], rows=dev[5])
    both = cc * ((1 - tt) * s + tt * s1)
    check(dw, db, cc * ((1 - tt) * s - tt * s1), both * (dz + 16 * U), "loss")
    term = torch.where(ok, cc * (tt * torch.nn.functional.softplus(-z) + (1 - tt) * torch.nn.functional.softplus(z)), 0.0)
    tol = (torch.where(ok, cc * dz, 0.0) + (16 + n + 2) * U * term + 4 * STEP).sum(0)
    assert bool(((loss.double().cpu() - term.sum(0)).abs() <= tol).all())
    dw, db, _ = tr.response_grad(dev[0], dev[1], dy.cuda(), dev[3], rows=dev[5])
    gr = dy.double() * s * s1
    check(dw, db, gr, gr.abs() * (dz + 12 * U), "responses")


@pytest.mark.parametrize("h", [8, 16])
def test_small_beside_large(tr, h):
    """Learners of small gradients beside learners of ordinary ones, and sets beside
    sets: each as precise as alone."""
    n, p = 500, 6
    g = torch.Generator().manual_seed(9)
    x = torch.rand(n, p, 32, generator=g).to(torch.bfloat16)
    w = torch.randn(p, h, 32, generator=g)
    dy = torch.randn(n, p, h, generator=g)
    scale = torch.ones(p, h)
    scale[1], scale[2, h // 2], scale[4, 0] = 2.0 ** -120, 2.0 ** -115, 0.0
    a = tr.response_grad(x.cuda(), w.cuda(), dy.cuda(), activation="none")
    b = tr.response_grad(x.cuda(), w.cuda(), (dy * scale).cuda(), activation="none")
    mag = torch.matmul(dy.double().abs().permute(1, 2, 0), x.double().transpose(0, 1))
    got, want = b[0].double().cpu(), a[0].double().cpu() * scale.double()[..., None]
    # either sum: one rounding a row
    assert bool(((got - want).abs() <= (2 * (n + 4) * U * mag) * scale.double()[..., None]).all())


@pytest.mark.parametrize("h", [8, 16])
@pytest.mark.parametrize("large", [1.0, 1e30, 2.0 ** 120])
def test_large_that_cancel(tr, large, h):
    """Large gradients of either sign beside small ones: sums of powers of two that
    come out exactly."""
    n, p = 64, 3
    x = torch.zeros(n, p, 32, dtype=torch.bfloat16)
    x[:, :, 0] = 1.0
    x[::2, :, 5] = 2.0
    x[63, :, 6] = 1.0
    dy = torch.zeros(n, p, h)
    dy[0], dy[1] = large, -large
    dy[63] = 2.0 ** -140
    dy[40, 1] = 2.0 ** -130 + 2.0 ** -149
    dw, db, _ = tr.response_grad(x.cuda(), torch.zeros(p, h, 32).cuda(), dy.cuda(), activation="none")
    dw, db = dw.cpu(), db.cpu()
    # (a sum may round the small ones away beside the large: place 0 and db)
    for got in (dw[..., 0], db):
        assert bool((got.abs() <= 2.0 ** -129).all())
    assert bool((dw[..., 5] == 2 * large).all()) and not dw[..., 7:].any()
    # (row 63 alone has place 6: beside large gradients a row's counts to 2^-133)
    assert bool(((dw[..., 6].double() - 2.0 ** -140).abs() <= 2.0 ** -133).all())
