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
