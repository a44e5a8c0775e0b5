"""Sums over very many rows (sc_lr_response_grad, sc_lr_loss): 32 bits hold a
bounded number of rows at a time, whatever the number of learners, so that the
error of a sum does not grow with the rows."""
import ctypes

import pytest
import torch

import surfcascade_amd as sc
from surfcascade_amd import _Samples, _WeakBank

U = 2.0 ** -24


@pytest.mark.parametrize("m,h,dtype", [(20000, 16, 2), (20000, 16, 0), (20000, 6, 1), (32768, 1, 0), (30000, 3, 2)])
def test_rows_are_cut_however_many_learners(m, h, dtype):
    """Learners enough to fill the chip alone: the rows of a call are cut all the
    same, and the workspace stays a few copies of the gradient."""
    L = sc.load_library()
    k = _WeakBank(m, h, 4096, 4096, None)
    n = ctypes.c_size_t()
    sets = m * h * 34
    for rows, least in ((8192, 0), (16385, 1), (100000, 1), (10**6, 1), (2**30, 1)):
        x = _Samples(4096, dtype, 4, 64, 128, 4096, rows)
        assert L.sc_lr_workspace(ctypes.byref(x), ctypes.byref(k), ctypes.byref(n)) == 0
        assert n.value >= least * sets * 4
        assert n.value <= max(sets * 4, 2**28) + sets * 8


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


def _equal_terms(p, r, seed):
    """64 samples whose values in a place are the same, and r numbers of them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(1, p, 32, generator=g).expand(64, p, 32).contiguous()
    rows = torch.randint(0, 64, (r,), generator=g, dtype=torch.int32)
    return x, rows


# (the largest a running sum of 2^11 terms of one sign can be off: a rounding of
# U a term; a result's last rounding, four waves' sums and their lanes' are a
# dozen more; a term: the loss' logarithm 3e-8 and 5 roundings, the gradient's
# slope 8 roundings, c (1 - t) and its product with the sample 2)
TERMS = 2048 + 12 + 10


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m,h,r", [("bf16", 5000, 16, 600000), ("f16", 5000, 16, 600000),
                                         ("f32", 5000, 16, 600000), ("bf16", 9000, 8, 600000),
                                         ("f32", 32768, 1, 400000), ("f16", 20000, 3, 400000),
                                         ("f32", 7, 2, 5000001)])
def test_equal_terms(tr, dtype, m, h, r):
    """w = 0, every weight 0.7, target 0: every row brings 0.7 log 2 and 0.35 x."""
    p = 4
    x, rows = _equal_terms(p, r, m)
    x = x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])
    patch = (torch.arange(m) % p).to(torch.int32)
    c = torch.full((64,), 0.7)
    loss, dw, db = tr.loss(x.cuda(), torch.zeros(m, h, 32, device="cuda"), torch.zeros(64, device="cuda"),
                           weight=c.cuda(), patch=patch.cuda(), rows=rows.cuda())
    weight = float(c[0]) * r
    want = weight * 0.6931471805599453
    assert float((loss.double() - want).abs().max()) <= TERMS * U * want
    assert float((db.double() - weight / 2).abs().max()) <= TERMS * U * weight / 2
    want = (x[0].double() * weight / 2)[patch.long()][:, None].cuda()  # [m, 1, 32]
    assert bool(((dw.double() - want).abs() <= TERMS * U * want).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m,h", [("bf16", 5000, 16), ("f32", 5000, 16), ("f16", 9000, 8), ("f32", 32768, 1)])
def test_response_gradient_of_many_rows(tr, dtype, m, h):
    """20001 rows of one dy and no activation, a seventh of them absent."""
    p, r = 4, 20001
    x, rows = _equal_terms(p, r, 3)
    x = x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])
    rows[::7] = -1
    there = int((rows >= 0).sum())
    patch = (torch.arange(m) % p).to(torch.int32)
    dy = torch.full((r, m, h), 0.3, device="cuda")
    dw, db, dres = tr.response_grad(x.cuda(), torch.zeros(m, h, 32, device="cuda"), dy, patch=patch.cuda(),
                                    rows=rows.cuda(), activation="none", residual="row", beta=0.5)
    g = 0.30000001192092896 * there  # (float32 0.3)
    assert float((db.double() - g).abs().max()) <= TERMS * U * g
    want = (x[0].double() * g)[patch.long()][:, None].cuda()
    assert bool(((dw.double() - want).abs() <= TERMS * U * want).all())
    d = 0.5 * 0.30000001192092896 * m * h
    assert float((dres.double() - d).abs().max()) <= 2 * U * d


@pytest.mark.gpu
def test_several_launches_in_a_graph(tr):
    """Rows over several launches, captured: each replay's results are its own
    inputs', with other calls of the trainer between them."""
    g = torch.Generator().manual_seed(5)
    x = torch.rand(64, 4, 32, generator=g).cuda()
    m, h, r = 40000, 16, 20000
    patch = (torch.arange(m) % 4).to(torch.int32).cuda()
    w = torch.randn(m, h, 32, generator=g).cuda()
    rows = torch.randint(0, 64, (r,), generator=g, dtype=torch.int32).cuda()
    t = torch.rand(64, generator=g).cuda()
    graph = torch.cuda.CUDAGraph()
    tr.loss(x, w, t, patch=patch, rows=rows)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = tr.loss(x, w, t, patch=patch, rows=rows)
    for k in range(3):
        t.copy_(torch.rand(64, generator=g))
        want = [v.clone() for v in tr.loss(x, w, t, patch=patch, rows=rows)]
        graph.replay()
        tr.loss(x, w, 1 - t, patch=patch, rows=rows)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
