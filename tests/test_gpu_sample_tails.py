"""Draws from long rows in which one place outweighs every other and the others
together still count (sc_sample): none of them may be lost in the unit of the
sums.  A place is off by half a unit, 2^-52 of the best weight: the n light places
before a border by n 2^-52 together, and the sum of all v that a random number is
a share of (of nearly 1) by v 2^-52, so a drawn place by (n + v) 2^-52 over one's
weight."""
import math

import pytest
import torch

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


def _row(v, best, low, dtype):
    s = torch.full((v,), low, dtype=DT[dtype], device="cuda")
    s[best] = 0.0
    return s


@pytest.mark.parametrize("v,low,dtype,temperature", [
    (2**26, -26.5, "f32", 1.0), (2**26, -26.5, "bf16", 1.0), (2**26 - 12345, -13.25, "f16", 0.5),
    (2**20 + 3, -30.0, "f32", 1.0), (40001, -30.0, "f32", 1.0), (32769, -3.0, "f32", 0.1)])
def test_light_places_are_drawn(tr, v, low, dtype, temperature):
    best = 777
    s = _row(v, best, low, dtype)
    w = math.exp(low / temperature)
    total = 1.0 + (v - 1) * w
    g = torch.Generator().manual_seed(v)
    # shares of the light places in order; the best place lies between two of them
    share = torch.cat([torch.rand(4000, generator=g, dtype=torch.float64), torch.tensor([1.0 - 2.0**-20], dtype=torch.float64)])
    place = (share * (v - 1)).floor()
    place = place[place > best]
    u = (1.0 + (place + 0.5) * w) / total       # the place-th light one, behind the best
    idx, kept = tr.sample(s, u.cuda(), temperature=temperature)
    assert int(kept) == v
    # u's and total's roundings: 4 units of 2^-53 each over a place's weight
    off = (place + v) * (2.0**-52 / w) + 8 * 2.0**-53 / w + 1
    assert bool(((idx.cpu().double() - (place + 1)).abs() <= off).all())
    before, _ = tr.sample(s, torch.tensor([0.25 * w / total, 0.5], dtype=torch.float64).cuda(), temperature=temperature)
    assert before.tolist() == [0, best]


@pytest.mark.parametrize("v,low", [(2**26, -26.5), (2**20 + 3, -30.0)])
def test_top_p_counts_the_light_places(tr, v, low):
    """top_p that takes half of what the light places bring keeps half of them."""
    s = _row(v, 12345, low, "f32")
    w = math.exp(low)
    total = 1.0 + (v - 1) * w
    half = (v - 1) // 2
    u = torch.tensor([0.0, 0.5, 1.0 - 2.0**-53], dtype=torch.float64).cuda()
    idx, kept = tr.sample(s, u, top_p=(1.0 + (half - 0.5) * w) / total)
    off = (half + v) * (2.0**-52 / w) + 8 * 2.0**-53 / w + 1
    assert abs(int(kept) - (1 + half)) <= off
    assert idx.tolist()[:2] == [0, 12345] and idx.tolist()[2] == int(kept) - 1
    idx, kept = tr.sample(s, u, top_k=v // 4, top_p=0.9999999999)
    assert abs(int(kept) - (v // 4)) <= 1e-10 * total / w + off  # (of top_k's mass: its last 1e-10)
    idx, kept = tr.sample(s, u, top_k=v // 4)
    assert int(kept) == v // 4 and idx.tolist()[2] == v // 4 - 1


@pytest.mark.parametrize("v", [8193, 40000, 2**20 + 1])
@pytest.mark.parametrize("temperature", [0.0, 1e-300, 1e-40, 1.0, 1e40, 1e300])
def test_sums_of_every_temperature(tr, v, temperature):
    """Weights that 32 bits cannot hold, beside infinite and lowest scores: the
    draws of the places that count are the definition's."""
    inf, low, most = math.inf, torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    g = torch.Generator().manual_seed(v)
    rows = torch.randn(5, v, generator=g)
    rows[1, ::2] = low
    rows[2, 5], rows[2, v - 9] = inf, inf
    rows[3] = 1e-42 * torch.randint(-3, 4, (v,), generator=g)  # denormals
    rows[4, 3] = most
    rows[4, ::7] = low
    u = torch.rand(5, 50, generator=g, dtype=torch.float64)
    from test_gpu_sample import reference
    for trim in (dict(), dict(top_k=9), dict(top_p=0.6)):
        want, wkept = reference(rows.double().numpy(), u.numpy(), temperature=temperature, **trim)
        idx, kept = tr.sample(rows.cuda(), u.cuda(), temperature=temperature, **trim)
        assert kept.tolist() == wkept.tolist()
        assert (idx.cpu().numpy() == want).all()
