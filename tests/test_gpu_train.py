"""Weak-learner responses, their gradient and the logistic loss over a sample
matrix (sc_lr_*), against the definitions in 64 bits.

Tolerances count roundings of U = 2^-24 (half a step of float32, relative):
* a dot of 32 products and a bias in any order: at most 33 roundings of values
  no larger than S = sum |x w| + |b|, so |dz| <= 34 U S;
* the sigmoid: its slope is at most 1/4; the exponential's argument is rounded
  twice (z * log2 e: |z| 2 U s(1-s) in the result) and the hardware's
  exponential, sum and reciprocal are good to 8 U together;
* a gradient sum of R terms g x: a row's g is off by its slope times dz and by
  8 roundings, and a sum of R terms in any order by at most R U sum |g x|.
"""
import math

import numpy as np
import pytest
import torch

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _make(n, p, m, h, dtype, seed, rows=0, picked=False, bias=True, absent=False):
    """CPU operands: descriptors of unit length, weights of a few units."""
    g = _rng(seed)
    x = torch.randn(n, p, 32, generator=g).abs()
    x = (x / x.norm(dim=2, keepdim=True).clamp_min(1e-6)).to(DT[dtype])
    w = 2 * torch.randn(*((m, h, 32) if h else (m, 32)), generator=g)
    b = torch.randn(*w.shape[:-1], generator=g) if bias else None
    patch = torch.randint(0, p, (m,), generator=g, dtype=torch.int32) if picked else None
    r = torch.randint(0, max(n, 1), (rows,), generator=g, dtype=torch.int32) if rows else None
    if absent and r is not None:
        bad = torch.tensor([-1, n, -2**31, 2**31 - 1], dtype=torch.int64).to(torch.int32)
        k = max(1, rows // 7)
        r[torch.randperm(rows, generator=g)[:k]] = bad[torch.randint(0, 4, (k,), generator=g)]
    if absent and patch is not None:
        patch[torch.randint(0, m, (max(1, m // 5),), generator=g)] = p
        patch[torch.randint(0, m, (max(1, m // 9),), generator=g)] = -1
    return x, w, b, patch, r


def _dev(t):
    return None if t is None else t.cuda()


class Ref:
    """The definitions in 64 bits: z, the absence mask, and S = sum |x w| + |b|."""

    def __init__(self, x, w, b, patch, rows):
        self.w3 = (w if w.dim() == 3 else w[:, None]).double()
        m, h = self.w3.shape[:2]
        n, p = x.shape[:2]
        rows = torch.arange(n) if rows is None else rows.long()
        patch = torch.arange(m) if patch is None else patch.long()
        self.row_ok = (rows >= 0) & (rows < n)
        self.patch_ok = (patch >= 0) & (patch < p)
        self.rows = torch.where(self.row_ok, rows, torch.zeros_like(rows))
        self.ok = (self.row_ok[:, None] & self.patch_ok[None, :])[:, :, None]
        if n == 0:
            self.x = torch.zeros(len(rows), m, 32, dtype=torch.float64)
        else:
            self.x = x.double()[self.rows][:, torch.where(self.patch_ok, patch, torch.zeros_like(patch))]
        b3 = torch.zeros(m, h, dtype=torch.float64) if b is None else b.double().reshape(m, h)
        self.z = torch.matmul(self.x.transpose(0, 1), self.w3.transpose(1, 2)).transpose(0, 1) + b3
        self.size = torch.matmul(self.x.abs().transpose(0, 1), self.w3.abs().transpose(1, 2)).transpose(0, 1) + b3.abs()

    def act(self, name):
        """(value, tolerance) of act(z)."""
        dz = 34 * U * self.size
        if name == "none":
            return self.z, dz
        s = torch.sigmoid(self.z)
        return s, 0.25 * dz + 4 * U * self.z.abs() * s * (1 - s) + 8 * U * s


def _near(got, want, tol, what=""):
    got = got.double().cpu().reshape(want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %g over a tolerance of %g" % (
        what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].max()), float(tol.reshape(-1)[bad.reshape(-1).nonzero()[0]]) if tol.dim() else float(tol))


SHAPES = [  # n, p, m, h (0: w is [m, 32]), rows, picked
    (1, 1, 1, 0, 0, False), (1, 608, 608, 0, 0, False), (7, 5, 5, 1, 0, False), (8, 9, 9, 2, 0, False),
    (9, 17, 33, 3, 0, True), (65, 16, 16, 4, 0, False), (64, 31, 31, 5, 100, False), (130, 40, 7, 8, 0, True),
    (33, 12, 12, 16, 33, False), (50, 10, 3, 17, 0, True), (20, 6, 6, 33, 41, False), (259, 64, 64, 0, 1, False),
    (1000, 20, 20, 0, 0, False), (40, 9, 9, 6, 0, False), (70, 21, 21, 7, 50, False), (48, 5, 5, 9, 0, False),
    (17, 4, 4, 15, 0, False), (129, 3, 11, 20, 64, True),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_response(tr, shape, dtype):
    n, p, m, h, rows, picked = shape
    x, w, b, patch, r = _make(n, p, m, h, dtype, 1, rows, picked, absent=True)
    ref = Ref(x, w, b, patch, r)
    R = len(ref.rows)
    g = _rng(5)
    for act in ("sigmoid", "none"):
        v, tol = ref.act(act)
        for kind in (None, "row", "full"):
            alpha, beta = (1.0, 1.0) if kind is None else (0.3, -0.7)
            a32, b32 = float(np.float32(alpha)), float(np.float32(beta))
            res = None if kind is None else torch.randn(R, generator=g) if kind == "row" else \
                torch.randn((R,) + tuple(w.shape[:-1]), generator=g)
            want = torch.where(ref.ok, a32 * v, torch.zeros_like(v))
            e = a32 * tol + 2 * U * want.abs()
            if res is not None:
                add = b32 * (res.double()[:, None, None] if kind == "row" else res.double().reshape(v.shape))
                want = want + add
                e = e + 2 * U * (add.abs() + want.abs())
            y = tr.response(_dev(x), _dev(w), _dev(b), patch=_dev(patch), rows=_dev(r), activation=act,
                            alpha=alpha, residual=_dev(res), beta=beta)
            assert y.shape == (R,) + tuple(w.shape[:-1]) and y.dtype == torch.float32
            _near(y, want, e, "%s %s" % (act, kind))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_response_grad(tr, shape, dtype):
    n, p, m, h, rows, picked = shape
    x, w, b, patch, r = _make(n, p, m, h, dtype, 2, rows, picked, absent=True)
    ref = Ref(x, w, b, patch, r)
    R = len(ref.rows)
    dy = torch.randn((R,) + tuple(w.shape[:-1]), generator=_rng(9))
    d = dy.double().reshape(ref.z.shape)
    for act, kind in (("sigmoid", "row"), ("none", "full"), ("sigmoid", None)):
        alpha, beta = 0.25, 0.75
        s = torch.sigmoid(ref.z)
        slope = s * (1 - s) if act == "sigmoid" else torch.ones_like(s)
        gr = torch.where(ref.ok, alpha * d * slope, torch.zeros_like(s))
        # |slope'| <= slope (s(1-s)|1-2s|); e^-|z| and its square carry |z| 2 U each
        eg = gr.abs() * (34 * U * ref.size + 8 * U * ref.z.abs() + 12 * U)
        _check_sums(tr.response_grad(_dev(x), _dev(w), _dev(dy), _dev(b), patch=_dev(patch), rows=_dev(r),
                                     activation=act, alpha=alpha, residual=kind, beta=beta)[:2], gr, eg, ref, R)
        dres = tr.response_grad(_dev(x), _dev(w), _dev(dy), _dev(b), patch=_dev(patch), rows=_dev(r),
                                activation=act, alpha=alpha, residual=kind, beta=beta)[2]
        if kind is None:
            assert dres is None
        elif kind == "full":
            assert dres.shape == dy.shape and torch.equal(dres.cpu(), dy * 0.75)
        else:
            assert dres.shape == (R,)
            want = beta * d.sum((1, 2))
            _near(dres, want, 2 * U * want.abs() + 1e-12 * d.abs().sum((1, 2)), "dres")


def _check_sums(got, gr, eg, ref, R):
    """dw and db against sum_r g x and sum_r g."""
    dw, db = got
    xx = torch.where(ref.ok, ref.x, torch.zeros_like(ref.x)).transpose(0, 1)  # [m, R, 32]
    gt = gr.permute(1, 2, 0)                                                  # [m, h, R]
    et = eg.permute(1, 2, 0)
    want = torch.matmul(gt, xx)
    tol = torch.matmul(et, xx.abs()) + (R + 2) * U * torch.matmul(gt.abs(), xx.abs()) + 1e-40
    assert dw.shape[:-1] == db.shape and dw.shape[-1] == 32
    _near(dw, want, tol, "dw")
    _near(db, gt.sum(2), et.sum(2) + (R + 2) * U * gt.abs().sum(2) + 1e-40, "db")


def _loss_ref(ref, t, c, n):
    """(loss, its tolerance, g, its tolerance)."""
    tt, cc = t.double()[ref.rows][:, None, None], c.double()[ref.rows][:, None, None]
    ok = ref.ok & (cc != 0)
    sp, sm = torch.nn.functional.softplus(ref.z), torch.nn.functional.softplus(-ref.z)
    term = torch.where(ok, cc * (tt * sm + (1 - tt) * sp), torch.zeros_like(sp))
    s, s1 = torch.sigmoid(ref.z), torch.sigmoid(-ref.z)
    g = torch.where(ok, cc * ((1 - tt) * s - tt * s1), torch.zeros_like(s))
    dz = 34 * U * ref.size
    both = torch.where(ok, cc.abs() * ((1 - tt) * s + tt * s1), torch.zeros_like(s))
    eg = both * (dz + 4 * U * ref.z.abs() + 16 * U)  # |ds| <= s |dz| on either side
    et = torch.where(ok, cc.abs() * (dz + 4 * U * ref.z.abs()), torch.zeros_like(s)) + 16 * U * term.abs()
    return term, et, g, eg


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss(tr, shape, dtype):
    n, p, m, h, rows, picked = shape
    x, w, b, patch, r = _make(n, p, m, h, dtype, 3, rows, picked, absent=True)
    g = _rng(11)
    for soft in (False, True):
        t = torch.rand(n, generator=g)
        t = t if soft else (t < 0.4).float()
        c = torch.rand(n, generator=g) + 0.1
        c[torch.rand(n, generator=g) < 0.2] = 0.0
        ref = Ref(x, w, b, patch, r)
        R = len(ref.rows)
        term, et, gr, eg = _loss_ref(ref, t, c, n)
        loss, dw, db = tr.loss(_dev(x), _dev(w), _dev(t), _dev(b), weight=_dev(c), patch=_dev(patch), rows=_dev(r))
        assert loss.shape == w.shape[:-1]
        _near(loss, term.sum(0), et.sum(0) + (R + 2) * U * term.abs().sum(0) + 1e-40, "loss")
        _check_sums((dw, db), gr, eg, ref, R)


def test_loss_without_weights_or_bias(tr):
    x, w, _, _, _ = _make(77, 19, 19, 0, "f32", 4)
    t = (torch.rand(77, generator=_rng(1)) < 0.5).float()
    ref = Ref(x, w, None, None, None)
    term, et, gr, eg = _loss_ref(ref, t, torch.ones(77), 77)
    loss, dw, db = tr.loss(_dev(x), _dev(w), _dev(t))
    _near(loss, term.sum(0), et.sum(0) + 79 * U * term.abs().sum(0), "loss")
    _check_sums((dw, db), gr, eg, ref, 77)


@pytest.mark.parametrize("dtype,h", [("f32", 1), ("bf16", 1), ("f16", 8), ("bf16", 16), ("bf16", 3), ("f32", 16)])
def test_loss_many_rows(tr, dtype, h):
    """Rows cut into chunks on the grid: the join of their partial sums.
    Random signs: the sums' own rounding stays far below the worst case of
    R roundings; a chunk's rows and its waves are summed one by one (at most
    2048 of them here) and the chunks in 64 bits."""
    n, p, m = 6001, 24, 24
    x, w, b, _, _ = _make(n, p, m, h, dtype, 5)
    t = (torch.rand(n, generator=_rng(2)) < 0.4).float()
    c = torch.rand(n, generator=_rng(3))
    ref = Ref(x, w, b, None, None)
    term, et, gr, eg = _loss_ref(ref, t, c, n)
    loss, dw, db = tr.loss(_dev(x), _dev(w), _dev(t), _dev(b), weight=_dev(c))
    _near(loss, term.sum(0), et.sum(0) + 2048 * U * term.sum(0), "loss")
    _check_sums((dw, db), gr, eg, ref, 2048)


def _one_hot(n, p, places):
    x = torch.zeros(n, p, 32)
    x[torch.arange(n), :, places] = 1.0
    return x


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h", [1, 2, 4, 7, 8, 16])
def test_places_and_sets_are_not_mixed(tr, h, dtype):
    """Descriptors of a single 1: every response is one weight, every gradient
    one row's sum, exactly."""
    n, p = 64, 6
    places = torch.arange(n) % 32
    x = _one_hot(n, p, places).to(DT[dtype])
    w = torch.randn(p, h, 32, generator=_rng(31))
    y = tr.response(x.cuda(), w.cuda(), activation="none").cpu()
    assert torch.equal(y, w[:, :, places].permute(2, 0, 1))
    dy = torch.randn(n, p, h, generator=_rng(32))
    dw, db, _ = tr.response_grad(x.cuda(), w.cuda(), dy.cuda(), activation="none")
    want = dy[:32].double() + dy[32:].double()  # rows k and 32 + k have place k
    _near(dw, want.permute(1, 2, 0), 2 * U * (dy[:32].abs() + dy[32:].abs()).double().permute(1, 2, 0), "dw")
    _near(db, dy.double().sum(0), 64 * U * dy.double().abs().sum(0), "db")


@pytest.mark.parametrize("h", [0, 2, 8])
def test_gradient_against_differences(tr, h):
    """dw and db against central differences of the loss itself, in 64 bits:
    the loss is smooth, so a step of 1e-4 leaves a third-derivative error of
    1e-8 c |x|^3 a row and 1e-12 / 1e-4 of rounding; 1e-5 of the sum of the
    weights covers both and the kernel's own roundings."""
    n, p, m = 41, 6, 6
    x, w, b, _, _ = _make(n, p, m, h, "f32", 6)
    t = torch.rand(n, generator=_rng(4))
    c = torch.rand(n, generator=_rng(5))
    _, dw, db = tr.loss(_dev(x), _dev(w), _dev(t), _dev(b), weight=_dev(c))

    def total(w_, b_):
        z = torch.matmul(x.double().transpose(0, 1), (w_ if w_.dim() == 3 else w_[:, None]).transpose(1, 2)).transpose(0, 1)
        z = z + b_.reshape(z.shape[1:])
        tt, cc = t.double()[:, None, None], c.double()[:, None, None]
        return float((cc * (torch.nn.functional.softplus(z) - tt * z)).sum())

    tol = 1e-5 * float(c.sum())
    wd, bd = w.double(), b.double()
    flat, dflat = wd.reshape(-1), dw.double().cpu().reshape(-1)
    for i in torch.randint(0, flat.numel(), (24,), generator=_rng(6)).tolist():
        keep = float(flat[i])
        flat[i] = keep + 1e-4
        up = total(wd, bd)
        flat[i] = keep - 1e-4
        down = total(wd, bd)
        flat[i] = keep
        assert abs((up - down) / 2e-4 - float(dflat[i])) <= tol
    bflat, dbf = bd.reshape(-1), db.double().cpu().reshape(-1)
    for i in range(min(8, bflat.numel())):
        keep = float(bflat[i])
        bflat[i] = keep + 1e-4
        up = total(wd, bd)
        bflat[i] = keep - 1e-4
        down = total(wd, bd)
        bflat[i] = keep
        assert abs((up - down) / 2e-4 - float(dbf[i])) <= tol


@pytest.mark.parametrize("h", [0, 8])
def test_response_grad_against_differences(tr, h):
    n, p, m = 23, 4, 4
    x, w, b, _, _ = _make(n, p, m, h, "f32", 7)
    dy = torch.randn((n,) + tuple(w.shape[:-1]), generator=_rng(8))
    dw, db, _ = tr.response_grad(_dev(x), _dev(w), _dev(dy), _dev(b), alpha=0.5)
    wd = w.double().reshape(m, -1, 32)

    def total(w_):
        z = torch.matmul(x.double().transpose(0, 1), w_.transpose(1, 2)).transpose(0, 1) + b.double().reshape(m, -1)
        return float((0.5 * torch.sigmoid(z) * dy.double().reshape(z.shape)).sum())

    flat, dflat = wd.reshape(-1), dw.double().cpu().reshape(-1)
    tol = 1e-5 * float(dy.abs().sum()) / m
    for i in torch.randint(0, flat.numel(), (24,), generator=_rng(9)).tolist():
        keep = float(flat[i])
        flat[i] = keep + 1e-4
        up = total(wd)
        flat[i] = keep - 1e-4
        down = total(wd)
        flat[i] = keep
        assert abs((up - down) / 2e-4 - float(dflat[i])) <= tol


@pytest.mark.parametrize("h", [1, 4, 16])
def test_what_is_absent_may_hold_anything(tr, h):
    """Rows of weight 0, rows out of range and learners out of range are not
    looked at: NaN and infinities there reach no result."""
    n, p, m = 40, 8, 8
    x, w, b, _, _ = _make(n, p, m, h, "f32", 8)
    bad = torch.tensor([3, 17, 39])
    good = torch.tensor([i for i in range(n) if i not in bad.tolist()])
    xb = x.clone()
    xb[bad] = float("nan")
    xb[17] = float("inf")
    t = (torch.rand(n, generator=_rng(2)) < 0.4).float()
    t[3] = float("nan")
    c = torch.rand(n, generator=_rng(3)) + 0.1
    c0 = c.clone()
    c0[bad] = 0.0
    got = tr.loss(_dev(xb), _dev(w), _dev(t), _dev(b), weight=_dev(c0))
    ref = Ref(x[good], w, b, None, None)
    term, et, gr, eg = _loss_ref(ref, t[good], c[good], len(good))
    _near(got[0], term.sum(0), et.sum(0) + 50 * U * term.sum(0), "loss")
    _check_sums(got[1:], gr, eg, ref, 50)
    # learners out of range beside a patch 0 of NaN
    xb = x.clone()
    xb[:, 0] = float("nan")
    patch = torch.arange(m, dtype=torch.int32)
    patch[0], patch[5] = -1, p
    loss, dw, db = tr.loss(_dev(xb), _dev(w), _dev(t.nan_to_num()), _dev(b), weight=_dev(c), patch=_dev(patch))
    for v in (loss, dw, db):
        assert torch.isfinite(v).all() and not v[0].any() and not v[5].any() and v[1].any()
    y = tr.response(_dev(xb), _dev(w), _dev(b), patch=_dev(patch))
    assert torch.isfinite(y).all() and not y[:, 0].any() and not y[:, 5].any()
    d = torch.ones(n, m, h).cuda()
    dw, db, _ = tr.response_grad(_dev(xb), _dev(w), d, _dev(b), patch=_dev(patch))
    assert torch.isfinite(dw).all() and not dw[0].any() and not db[5].any()


@pytest.mark.parametrize("h", [1, 16])
def test_values_out_of_range_show(tr, h):
    """A NaN or an infinity in a row that counts is not hidden."""
    x, w, b, _, _ = _make(20, 3, 3, h, "f32", 9)
    x[7, 1, 5] = float("nan")
    t = torch.zeros(20)
    y = tr.response(_dev(x), _dev(w), _dev(b))
    assert torch.isnan(y[7, 1]).all() and torch.isfinite(y[:, 0]).all() and torch.isfinite(y[6]).all()
    loss, dw, db = tr.loss(_dev(x), _dev(w), _dev(t), _dev(b))
    assert torch.isnan(loss[1]).all() and torch.isnan(db[1]).all() and torch.isnan(dw[1]).all()
    assert torch.isfinite(loss[0]).all() and torch.isfinite(dw[2]).all()


def test_saturated_learners(tr):
    """|z| of hundreds: the response is 0 or 1, the loss |z| where it is wrong."""
    x = torch.zeros(4, 1, 32)
    x[:, 0, 0] = torch.tensor([1.0, 1.0, -1.0, -1.0])
    w = torch.zeros(1, 32)
    w[0, 0] = 500.0
    t = torch.tensor([1.0, 0.0, 1.0, 0.0])
    y = tr.response(x.cuda(), w.cuda())
    assert y.cpu().flatten().tolist() == [1.0, 1.0, 0.0, 0.0]
    loss, dw, db = tr.loss(x.cuda(), w.cuda(), t.cuda())
    assert loss.item() == 1000.0 and db.item() == 0.0 and dw[0, 0].item() == 2.0
    dw, db, _ = tr.response_grad(x.cuda(), w.cuda(), torch.ones(4, 1).cuda())
    assert not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strides_and_alignment(tr, dtype):
    """Samples at any element, any stride between them; results and residuals
    in wider buffers, whose other values stay as they were."""
    n, p, m, h = 37, 11, 11, 3
    x, w, b, _, _ = _make(n, p, m, h, dtype, 10)
    wide = torch.full((n * (p * 32 + 5) + 64,), 7.0, dtype=DT[dtype]).cuda()
    xs = wide[3:].as_strided((n, p, 32), (p * 32 + 5, 32, 1))
    xs.copy_(x)
    plain = tr.response(_dev(x), _dev(w), _dev(b))
    assert torch.equal(tr.response(xs, _dev(w), _dev(b)), plain)
    big = torch.full((n, m * h + 4), 9.0).cuda()
    out = big[:, 1:1 + m * h].unflatten(1, (m, h))
    assert tr.response(xs, _dev(w), _dev(b), out=out) is out
    assert torch.equal(out, plain) and (big[:, 0] == 9).all() and (big[:, 1 + m * h:] == 9).all()
    res = torch.randn(n, m * h + 4, generator=_rng(1)).cuda()
    ref = tr.response(xs, _dev(w), _dev(b), alpha=0.5, residual=res[:, 2:2 + m * h].contiguous(), beta=0.5)
    got = tr.response(xs, _dev(w), _dev(b), alpha=0.5, residual=res[:, 2:2 + m * h], beta=0.5)
    assert torch.equal(got, ref)
    rowres = torch.randn(n, 3, generator=_rng(2)).cuda()
    assert torch.equal(tr.response(xs, _dev(w), _dev(b), residual=rowres[:, 1]),
                       tr.response(xs, _dev(w), _dev(b), residual=rowres[:, 1].contiguous()))
    # in place over the residual
    run = res[:, 2:2 + m * h].contiguous()
    assert torch.equal(tr.response(xs, _dev(w), _dev(b), alpha=0.5, residual=run, beta=0.5, out=run).view(ref.shape), ref)
    t = (torch.rand(n, generator=_rng(4)) < 0.5).float().cuda()
    for u, v in zip(tr.loss(xs, _dev(w), t, _dev(b)), tr.loss(_dev(x), _dev(w), t, _dev(b))):
        assert torch.equal(u, v)
    dy = torch.randn(n, m * h + 7, generator=_rng(3)).cuda()
    for u, v in zip(tr.response_grad(xs, _dev(w), dy[:, 3:3 + m * h], _dev(b), residual="full"),
                    tr.response_grad(xs, _dev(w), dy[:, 3:3 + m * h].contiguous(), _dev(b), residual="full")):
        assert torch.equal(u, v)


def test_empty_sizes(tr):
    f = dict(device="cuda")
    x, w = torch.zeros(0, 5, 32, **f), torch.randn(5, 2, 32, **f)
    assert tr.response(x, w).shape == (0, 5, 2)
    for v in tr.loss(x, w, torch.zeros(0, **f)):
        assert not v.any()
    for v in tr.response_grad(x, w, torch.zeros(0, 5, 2, **f))[:2]:
        assert not v.any()
    # rows of an empty matrix are all absent
    rows = torch.tensor([0, 1, -1], dtype=torch.int32, **f)
    res = torch.arange(3, **f).float()
    assert torch.equal(tr.response(x, w, rows=rows, residual=res, beta=2.0)[:, 3, 1], 2 * res)
    for v in tr.loss(x, w, torch.zeros(0, **f), rows=rows):
        assert not v.any()
    x = torch.randn(4, 5, 32, **f)
    none = torch.zeros(0, dtype=torch.int32, **f)
    assert tr.response(x, w, rows=none).shape == (0, 5, 2)
    for v in tr.loss(x, w, torch.zeros(4, **f), rows=none):
        assert not v.any()
    w0 = torch.zeros(0, 2, 32, **f)
    assert tr.response(x, w0).shape == (4, 0, 2)
    assert tr.loss(x, w0, torch.zeros(4, **f))[0].shape == (0, 2)
    dw, db, dres = tr.response_grad(x, w0, torch.zeros(4, 0, 2, **f), residual="row")
    assert dw.shape == (0, 2, 32) and dres.shape == (4,) and not dres.any()


def test_offsets_past_32_bits(tr):
    """Samples more than 2^31 elements apart."""
    ld = 2**30 + 3 * 32
    buf = torch.empty(2 * ld + 3 * 32, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, 3, 32), (ld, 32, 1))
    xc, w, b, _, _ = _make(3, 3, 3, 2, "bf16", 11)
    x.copy_(xc)
    rows = torch.tensor([2, 0, 1, 2], dtype=torch.int32).cuda()
    assert torch.equal(tr.response(x, _dev(w), _dev(b), rows=rows), tr.response(_dev(xc), _dev(w), _dev(b), rows=rows))
    t = torch.tensor([1.0, 0.0, 1.0]).cuda()
    for u, v in zip(tr.loss(x, _dev(w), t, rows=rows), tr.loss(_dev(xc), _dev(w), t, rows=rows)):
        assert torch.equal(u, v)


def test_same_call_same_bits(tr):
    x, w, b, _, r = _make(3000, 40, 40, 2, "f32", 12, rows=5000)
    t = (torch.rand(3000, generator=_rng(2)) < 0.4).float().cuda()
    first = tr.loss(_dev(x), _dev(w), t, _dev(b), rows=_dev(r))
    for _ in range(3):
        for u, v in zip(first, tr.loss(_dev(x), _dev(w), t, _dev(b), rows=_dev(r))):
            assert torch.equal(u, v)


def test_refused_tensors(tr):
    x, w, b, _, _ = _make(6, 4, 4, 0, "f32", 13)
    X, W, B = x.cuda(), w.cuda(), b.cuda()
    t = torch.zeros(6).cuda()
    for bad in (lambda: tr.response(x, W), lambda: tr.response(X, w), lambda: tr.response(X.double(), W),
                lambda: tr.response(X, W.half()), lambda: tr.response(X[:, :, :16], W),
                lambda: tr.response(X.transpose(1, 2).contiguous().transpose(1, 2), W),
                lambda: tr.response(X[:, ::2], W), lambda: tr.response(X.expand(2, 6, 4, 32)[0][:1].expand(6, 4, 32), W),
                lambda: tr.response(X, torch.cat([W, W])), lambda: tr.response(X, W, B[:3]),
                lambda: tr.response(X, W, patch=torch.zeros(4).cuda()),
                lambda: tr.response(X, W, rows=torch.zeros(4, dtype=torch.int64).cuda()),
                lambda: tr.response(X, W, residual=torch.zeros(5).cuda()),
                lambda: tr.response(X, W, residual=torch.zeros(6, 3).cuda()),
                lambda: tr.response(X, W, residual=torch.zeros(4, 6).cuda().t()),
                lambda: tr.response(X, W, out=torch.zeros(6, 4)),
                lambda: tr.response(X, W, out=torch.zeros(6, 4, dtype=torch.float64).cuda()),
                lambda: tr.response(X, W.t().contiguous().t()),
                lambda: tr.loss(X, W, t[:5]), lambda: tr.loss(X, W, t.double()), lambda: tr.loss(X, W, t, weight=t[:3]),
                lambda: tr.response_grad(X, W, torch.zeros(5, 4).cuda())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(KeyError):
        tr.response(X, W, activation="tanh")


def test_host_pointers_and_small_workspaces(tr):
    """What the C ABI itself refuses on a GPU machine."""
    import ctypes

    from surfcascade_amd.train import _Samples, _WeakBank
    L = sc.load_library()
    x, w, b, _, _ = _make(9000, 4, 4, 0, "f32", 14)
    X, W, T = x.cuda(), w.cuda(), torch.zeros(9000).cuda()
    loss, dw, db = torch.zeros(4).cuda(), torch.zeros(4, 32).cuda(), torch.zeros(4).cuda()

    def call(xp=None, wp=None, tp=None, ws=None, n=0):
        s = _Samples(xp or X.data_ptr(), 0, 4, 9000, 128, None, 0)
        k = _WeakBank(4, 1, None, wp or W.data_ptr(), None)
        return L.sc_lr_loss(tr._h, ctypes.byref(s), ctypes.byref(k), tp or T.data_ptr(), None, loss.data_ptr(),
                            dw.data_ptr(), db.data_ptr(), ws, n)

    assert call() == 0  # the trainer's own workspace
    tr.synchronize()
    own = dw.clone()
    assert call(xp=x.data_ptr()) == -1 and b"samples" in L.sc_last_error()
    assert call(wp=w.data_ptr()) == -1 and call(tp=x.data_ptr()) == -1
    assert call(xp=X.data_ptr() + 2) == -1 and b"aligned" in L.sc_last_error()
    ws = torch.empty(1 << 20, dtype=torch.uint8).cuda()
    assert call(ws=ws.data_ptr(), n=64) == -6
    assert call(ws=ws.data_ptr() + 8, n=(1 << 20) - 8) == -1 and b"16" in L.sc_last_error()
    assert call(ws=x.data_ptr(), n=1 << 20) == -1
    assert call(ws=ws.data_ptr(), n=1 << 20) == 0
    tr.synchronize()
    assert torch.equal(own, dw)


def test_other_streams(tr):
    """A call runs on torch's current stream: behind the work that fills its
    operands, ahead of the work that reads its results."""
    x, w, b, _, _ = _make(2000, 64, 64, 0, "f32", 15)
    want = tr.response(_dev(x), _dev(w), _dev(b))
    W, B, src = _dev(w), _dev(b), _dev(x)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2, s1):
        with torch.cuda.stream(s):
            X = torch.zeros_like(src)
            torch.cuda._sleep(2000000)
            X.copy_(src)
            y = tr.response(X, W, B)
            z = y.clone()
        s.synchronize()
        assert torch.equal(z, want)
    assert torch.equal(tr.response(src, W, B), want)


def test_captured_and_replayed():
    """Responses, loss and draws in one graph; two graphs of one trainer, their
    replays and eager calls in turn; inputs change between replays."""
    tr = sc.Trainer()
    x, w, b, _, _ = _make(5000, 12, 12, 2, "f32", 16)
    X, W, B = _dev(x), _dev(w), _dev(b)
    t = (torch.rand(5000, generator=_rng(2)) < 0.4).float().cuda()
    sco = torch.randn(5000, generator=_rng(3)).cuda()
    u = torch.rand(777, generator=_rng(4), dtype=torch.float64).cuda()

    def step(score):
        idx, kept = tr.sample(score, u, temperature=0.8, top_p=0.9)
        loss, dw, db = tr.loss(X, W, t, B, rows=idx)
        y = tr.response(X, W, B, rows=idx)
        return idx, kept, loss, dw, db, y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sco)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, ins, outs = [], [], []
    for k in range(2):
        s = torch.zeros_like(sco)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(s)
        graphs.append(g)
        ins.append(s)
        outs.append(o)
    for k in range(6):
        score = sco.roll(k) * (1 + 0.1 * k)
        want = [v.clone() for v in step(score)]
        ins[k % 2].copy_(score)
        graphs[k % 2].replay()
        other = step(sco)  # eager work behind the replay
        torch.cuda.synchronize()
        for a, e in zip(outs[k % 2], want):
            assert torch.equal(a, e)
        assert torch.equal(other[0], step(sco)[0])


def test_capture_needs_its_own_workspace():
    """A captured C call that needs a workspace and brings none is refused."""
    import ctypes

    from surfcascade_amd.train import _Samples, _WeakBank
    L = sc.load_library()
    tr = sc.Trainer()
    X, W, T = torch.rand(9000, 4, 32).cuda(), torch.rand(4, 32).cuda(), torch.zeros(9000).cuda()
    o = torch.zeros(4 * 34).cuda()
    s, k = _Samples(X.data_ptr(), 0, 4, 9000, 128, None, 0), _WeakBank(4, 1, None, W.data_ptr(), None)
    y = tr.response(X, W)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tr._follow()
        rc = L.sc_lr_loss(tr._h, ctypes.byref(s), ctypes.byref(k), T.data_ptr(), None, o.data_ptr(), o.data_ptr() + 16,
                          o.data_ptr() + 600 - 600 % 16, None, 0)
        msg = L.sc_last_error()
        y2 = tr.response(X, W)
    assert rc == -1 and b"workspace" in msg
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y2)


# -- with the miner and the models ------------------------------------------------

def test_stage_responses_agree_with_the_miner(tr):
    """A trained stage's weak classifiers over mined descriptors: the mean of
    their responses is the stage score the cascade kernels give the window
    (GentleAdaboost::Predict2)."""
    from conftest import FACE_CFG
    from surfcascade_amd import synth
    casc = sc.CascadeClassifier()
    assert sc.Model(FACE_CFG).Load(casc) == 0
    stage = casc.stage_classifiers[0]
    miner = sc.Miner(None)
    img = torch.from_numpy(synth.make_frame(240, 180, 3)).cuda()
    feat = torch.zeros(256, miner.n_patches, 32, device="cuda")
    _, total = miner.mine_device(img, 256, feat)
    n = min(total, 256)
    w, b, patch = tr.bank(stage.weak_classifiers)
    y = tr.response(feat[:n], w, b, patch=patch)
    assert y.shape == (n, len(stage.weak_classifiers))
    f = feat[:n].double().cpu()
    want = torch.stack([torch.sigmoid(f[:, k.patch_index] @ torch.tensor(k.w[:32]).double() + float(k.w[32]) * k.bias)
                        for k in stage.weak_classifiers], 1)
    size = torch.stack([f[:, k.patch_index].abs() @ torch.tensor(np.abs(k.w[:32])).double() + abs(float(k.w[32]) * k.bias)
                        for k in stage.weak_classifiers], 1)
    _near(y, want, 0.25 * 34 * U * size + 4 * U * size + 8 * U, "stage")
    # against the cascade kernels' own stage score: its weak outputs and their
    # mean are rounded to float32 too
    one = sc.Model.parse(synth.write_cfg(synth.cascade_tree(
        np.array([len(stage.weak_classifiers)]), np.array([-1.0], np.float32),
        np.array([k.patch_index for k in stage.weak_classifiers]),
        np.stack([k.w for k in stage.weak_classifiers]), np.array([k.bias for k in stage.weak_classifiers]))))
    wins, total2 = sc.Miner(one).mine_device(img, 256)
    assert total2 == total
    mean = y.double().mean(1).cpu().numpy()
    assert np.abs(wins["score"][:n] - mean).max() <= 1e-5


def test_boosting_round(tr):
    """Mine, resample, fit and score, as a boosting round uses them: the loss
    falls the way the same steps in 64 bits say, and the running score is the
    mean of the fitted learners."""
    from surfcascade_amd import synth
    miner = sc.Miner(None)
    frames = torch.from_numpy(synth.make_frames(320, 240, 2)).cuda()
    n = 512
    feat = torch.zeros(n, miner.n_patches, 32, device="cuda")
    _, counts = miner.mine_batch_device(frames, n, feat)
    assert counts.sum() >= n
    g = _rng(21)
    target = (torch.rand(n, generator=g) < 0.5).float()
    logw = torch.randn(n, generator=g)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    rows, kept = tr.sample(logw.cuda(), u.cuda(), top_p=0.99)
    assert 0 < int(kept) <= n and rows.shape == (n,)
    m = miner.n_patches
    w, b = torch.zeros(m, 32, device="cuda"), torch.zeros(m, device="cuda")
    wd, bd = w.double().cpu(), b.double().cpu()
    f = feat.double().cpu()[rows.cpu().long()]
    t = target.double()[rows.cpu().long()][:, None]
    lr = 1e-2
    for _ in range(4):
        loss, dw, db = tr.loss(feat, w, target.cuda(), b, rows=rows)
        z = torch.matmul(f.transpose(0, 1), wd[:, :, None])[:, :, 0].t() + bd
        want = (torch.nn.functional.softplus(z) - t * z).sum(0)
        assert torch.allclose(loss.double().cpu(), want, rtol=1e-4, atol=0)
        gd = torch.sigmoid(z) - t
        wd = wd - lr * torch.matmul(gd.t()[:, None, :], f.transpose(0, 1))[:, 0]
        bd = bd - lr * gd.sum(0)
        w, b = w - lr * dw, b - lr * db
    score = torch.zeros(n, device="cuda")
    pick = torch.tensor([5, 100, 607], dtype=torch.int32, device="cuda")
    for k, j in enumerate(pick.tolist(), 1):
        y = tr.response(feat, w[j:j + 1], b[j:j + 1], patch=pick[k - 1:k], alpha=1.0 / k, residual=score,
                        beta=1.0 - 1.0 / k)
        score = y[:, 0].contiguous()
    fa = feat.double().cpu()
    want = torch.stack([torch.sigmoid(fa[:, j] @ wd[j] + bd[j]) for j in pick.tolist()], 1).mean(1)
    assert torch.allclose(score.double().cpu(), want, rtol=0, atol=1e-4)


def test_workspace_order_around_a_capture():
    """A call on a third stream, after one was captured on a second, waits for
    the first stream's call: both use the trainer's workspace."""
    tr = sc.Trainer()
    X, W, T = torch.rand(9000, 4, 32).cuda(), torch.rand(4, 32).cuda(), torch.zeros(9000).cuda()
    want = [v.clone() for v in tr.loss(X, W, T)]
    a, b, c = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    g, end = torch.cuda.CUDAGraph(), torch.cuda.Event()
    with torch.cuda.stream(a):
        torch.cuda._sleep(100_000_000)
        busy = torch.cuda.Event()
        busy.record()
        first = tr.loss(X, W, T)
    with torch.cuda.stream(b):
        g.capture_begin()
        y = tr.response(X, W)
        g.capture_end()
    with torch.cuda.stream(c):
        second = tr.loss(X, W, T)
        end.record()
        done = end.query()
        assert not (done and not busy.query())
    torch.cuda.synchronize()
    for got in (first, second):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, tr.response(X, W))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("h", [1, 16])
def test_infinite_weights(tr, h, dtype):
    """z = -inf: a sigmoid of 0 and, for target 0, gradients of 0 (the loss has a
    0 * inf, also in its formula)."""
    x = (0.25 + torch.rand(70, 3, 32, generator=_rng(5))).to(DT[dtype]).cuda()
    w = torch.zeros(3, h, 32, device="cuda")
    w[1, h // 2, 7] = -math.inf
    y = tr.response(x, w)
    assert bool((y[:, 1, h // 2] == 0).all()) and not bool(torch.isnan(y).any())
    dw, db, _ = tr.response_grad(x, w, torch.ones_like(y))
    assert bool((dw[1, h // 2] == 0).all()) and float(db[1, h // 2]) == 0
    _, dw, db = tr.loss(x, w, torch.zeros(70, device="cuda"))
    assert bool((dw[1, h // 2] == 0).all()) and float(db[1, h // 2]) == 0
    assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())


def test_no_rows_of_very_many_learners(tr):
    """2^25 learner sets, whose zeros are more workgroups' than a grid has."""
    w = torch.ones(2**20, 32, 32, device="cuda")
    patch = torch.zeros(2**20, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = tr.loss(torch.rand(4, 2, 32, device="cuda"), w, torch.zeros(4, device="cuda"), patch=patch, rows=none)
    for v in out:
        assert not bool(v.any())


def test_operands_that_want_gradients_are_refused(tr):
    """Nothing connects a result to its operands, so it must not look as if."""
    x, w, b, _, _ = _make(9, 3, 3, 2, "f32", 1)
    X, W, B = x.cuda(), w.cuda(), b.cuda()
    t, u = torch.zeros(9, device="cuda"), torch.rand(4, dtype=torch.float64, device="cuda")
    leaf = W.clone().requires_grad_()
    for call in (lambda w: tr.response(X, w, B), lambda w: tr.response(X, W, w[..., 0].contiguous()),
                 lambda w: tr.response(X, W, B, residual=w[:, :, 0].sum().expand(9, 3, 2).contiguous()),
                 lambda w: tr.loss(X, w, t, B), lambda w: tr.response_grad(X, w, torch.ones(9, 3, 2, device="cuda")),
                 lambda w: tr.sample(w[0, 0], u)):
        with pytest.raises(ValueError, match="autograd"):
            call(leaf)
        call(W)
        with torch.no_grad():
            call(leaf)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("h,m", [(5, 2), (6, 7), (8, 1), (8, 9), (7, 16)])
def test_neighbouring_learners_stay_apart(tr, h, m, dtype):
    """A NaN in one learner's descriptors, weights or dy is that learner's alone;
    an absent patch's learner is zero whatever stands in the samples."""
    n, p = 67, 20
    x, w, b, _, _ = _make(n, p, m, h, dtype, 40 + m)
    patch = torch.arange(m, dtype=torch.int32) + 2
    dy = torch.randn(n, m, h, generator=_rng(m))
    t = (torch.rand(n, generator=_rng(h)) < 0.5).float()

    def run(x, w, dy, patch):
        dw, db, dres = tr.response_grad(x.cuda(), w.cuda(), dy.cuda(), b.cuda(), patch=patch.cuda(), residual="full")
        return [v.cpu() for v in (dw, db, dres.permute(1, 0, 2), *tr.loss(x.cuda(), w.cuda(), t.cuda(), b.cuda(),
                                                                          patch=patch.cuda()))]

    clean = run(x, w, dy, patch)
    assert all(bool(torch.isfinite(v).all()) for v in clean)
    for bad in range(m):
        xs, ws, ds, ps = x.clone(), w.clone(), dy.clone(), patch.clone()
        xs[33, bad + 2, 5] = math.nan
        for got, want in zip(run(xs, w, dy, patch), clean):  # (dres does not read the samples)
            keep = torch.arange(m) != bad
            assert torch.equal(got[keep], want[keep])
        ws[bad, h - 1] = math.nan
        got = run(x, ws, dy, patch)
        assert bool(torch.isnan(got[1][bad, h - 1])) and bool(torch.isnan(got[3][bad, h - 1]))
        for g, c in zip(got, clean):
            keep = torch.ones(m, h, dtype=torch.bool)
            keep[bad, h - 1] = False
            if g.dim() == 3 and g.shape[1] == n:
                continue
            assert torch.equal(g[keep], c[keep])
        ds[12, bad, 0] = math.nan
        got = run(x, w, ds, patch)
        assert bool(torch.isnan(got[1][bad, 0]))
        keep = torch.ones(m, h, dtype=torch.bool)
        keep[bad, 0] = False
        assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
        ps[bad] = p + 3
        xs = x.clone()
        xs[:, 0] = math.nan  # (nobody's patch)
        for k, (g, c) in enumerate(zip(run(xs, w, dy, ps), clean)):
            keep = torch.arange(m) != bad
            assert torch.equal(g[keep], c[keep])
            assert k == 2 or not bool(g[bad].any())
