"""Weights and biases near the largest float32 (3.4e38): finite operands whose
definition is finite give finite results.  Tolerances count roundings of
U = 2^-24: a bias passes through no product (one rounding in the loss, one in
the sum of one row that is not 0, the rest exact)."""
import pytest
import torch

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h", [1, 3, 6, 8, 16])
def test_largest_biases(tr, h, dtype):
    """z = +-3e38: a response of 0 or 1, no slope, and for the wrong target a loss
    of c |z|, whatever units the exponential has."""
    n, m = 40, 3
    x = torch.zeros(n, m, 32).to(DT[dtype])
    x[:, :, 0] = 1.0
    b = torch.zeros(m, h)
    b[1], b[2] = 3.0e38, -3.0e38
    w = torch.zeros(m, h, 32)
    t, c = torch.zeros(n), torch.zeros(n)
    t[11] = 1.0
    c[[11, 30]] = 2.0 ** -9
    dev = [v.cuda() for v in (x, w, t, b, c)]
    y = tr.response(dev[0], dev[1], dev[3]).cpu()
    assert bool((y[:, 1] == 1).all()) and bool((y[:, 2] == 0).all())
    dw, db, _ = tr.response_grad(dev[0], dev[1], torch.ones(n, m, h, device="cuda"), dev[3])
    assert not dw[1:].any() and not db[1:].any()
    loss, dw, db = (v.double().cpu() for v in tr.loss(dev[0], dev[1], dev[2], dev[3], weight=dev[4]))
    z = 2.0 ** -9 * b[1:].double().abs()
    assert bool(((loss[1:] - z).abs() <= 2 * U * z).all())
    # row 30 (target 0) is wrong under +3e38, row 11 (target 1) under -3e38
    for k, g in ((1, 2.0 ** -9), (2, -(2.0 ** -9))):
        assert bool((db[k] == g).all()) and bool((dw[k, :, 0] == g).all()) and not dw[k, :, 1:].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h", [1, 3, 6, 8, 16])
def test_largest_weights(tr, h, dtype):
    """A weight of 3e38 beside a sample's 0 brings nothing, beside 2^-126 some 3.5."""
    n, m = 35, 4
    x = torch.zeros(n, m, 32).to(DT[dtype])
    tiny = 2.0 ** -24 if dtype == "f16" else 2.0 ** -126
    x[20, :, 7] = tiny
    w = torch.zeros(m, h, 32)
    w[:, :, 7] = 3.0e38 if dtype != "f16" else 3.0e38 * 2.0 ** -103
    w[2, :, 9] = -3.2e38  # (every sample: 0)
    z = float(w[0, 0, 7].double()) * tiny
    y = tr.response(x.cuda(), w.cuda(), activation="none").double().cpu()
    want = torch.zeros(n, m, h, dtype=torch.float64)
    want[20] = z
    assert bool(((y - want).abs() <= U * want).all())
    dy = torch.ones(n, m, h)
    _, db, _ = tr.response_grad(x.cuda(), w.cuda(), dy.cuda())
    s = torch.sigmoid(torch.tensor(z, dtype=torch.float64))
    g = float(s * (1 - s))
    total = (n - 1) * 0.25 + g
    # a row's slope: z to one rounding, its exponential 4 z roundings, 12 besides
    assert float((db.double().cpu() - total).abs().max()) <= (g * (5 * z + 12) + (n + 2 + 12) * total) * U
    loss, _, db = tr.loss(x.cuda(), w.cuda(), torch.zeros(n).cuda())
    total = (n - 1) * 0.6931471805599453 + float(torch.nn.functional.softplus(torch.tensor(z, dtype=torch.float64)))
    assert float((loss.double().cpu() - total).abs().max()) <= (5 * z + (n + 2 + 16) * total) * U
    total = (n - 1) * 0.5 + float(s)
    assert float((db.double().cpu() - total).abs().max()) <= (5 * z + (n + 2 + 16) * total) * U
