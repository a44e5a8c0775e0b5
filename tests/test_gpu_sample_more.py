"""Draws from scores (sc_sample) where test_gpu_sample.py's sizes do not go: more
long rows than share a workspace, very many draws of one workgroup's rows, numbers
outside a C int."""
import pytest
import torch

import surfcascade_amd as sc
from test_gpu_sample import DT, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


@pytest.mark.parametrize("top_k", [-1, -2**31, -2**31 - 1, -2**32, -2**40])
def test_top_k_below_zero(tr, top_k):
    scores, u = torch.zeros(2, 9).cuda(), torch.zeros(2, 3, dtype=torch.float64).cuda()
    with pytest.raises(sc.SurfCascadeError) as e:
        tr.sample(scores, u, top_k=top_k)
    assert e.value.code == -1


def test_top_k_above_a_c_int(tr):
    scores, u = torch.zeros(1, 9).cuda(), torch.full((1, 1), 0.99, dtype=torch.float64).cuda()
    idx, kept = tr.sample(scores, u, top_k=2**40)
    assert int(idx) == 8 and int(kept) == 9


def _rows(b, v, s, seed, dtype="f32"):
    g = torch.Generator().manual_seed(seed)
    return (2 * torch.randn(b, v, generator=g)).to(DT[dtype]), torch.rand(b, s, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("trim", [dict(), dict(top_p=0.9), dict(top_k=8500, top_p=0.8, min_p=1e-3)], ids=str)
def test_more_long_rows_than_share_a_workspace(tr, trim, dtype):
    """512 rows cut over many workgroups share the workspace at a time; 1100 rows of
    their own lengths, scores, numbers and results in wider buffers, take three."""
    b, v, s = 1100, 8301, 6
    scores, u = _rows(b, v, s, 3, dtype)
    lens = torch.randint(0, v + 1, (b,), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    lens[[0, 511, 512, 1023, 1024]] = v
    lens[[1, 513]] = 0
    wide = torch.full((b, v + 9), float("inf"), dtype=DT[dtype])
    wide[:, 3:v + 3] = scores
    wu = torch.full((b, s + 5), 0.5, dtype=torch.float64)
    wu[:, 2:s + 2] = u
    want, wkept = reference(scores.double().numpy(), u.numpy(), lens=lens.numpy(), **trim)
    idx, kept = tr.sample(wide.cuda()[:, 3:v + 3], wu.cuda()[:, 2:s + 2], lens=lens.cuda(), **trim)
    assert (kept.cpu().numpy() == wkept).all()
    assert (idx.cpu().numpy() == want).all()


@pytest.mark.parametrize("b,v,s,trim", [
    (1, 200, 2**20, dict()), (1, 960, 2**20, dict(top_p=0.97)), (3, 960, 70001, dict(top_k=100)),
    (1, 4000, 2**18 + 3, dict(min_p=0.01)), (1, 8192, 2**19, dict()), (2, 8192, 2**17, dict(top_k=3000, top_p=0.9)),
    (1, 20011, 2**18, dict(top_k=2000, top_p=0.95)), (1, 12000, 2**18 + 1, dict(top_k=700)),
    (9, 30000, 2**15, dict(top_k=5000))], ids=str)
def test_very_many_draws_of_one_workgroup(tr, b, v, s, trim):
    scores, u = _rows(b, v, s, v + s)
    want, wkept = reference(scores.double().numpy(), u.numpy(), **trim)
    idx, kept = tr.sample(scores.cuda(), u.cuda(), **trim)
    assert (kept.cpu().numpy() == wkept).all()
    assert (idx.cpu().numpy() == want).all()
