"""Calls of one trainer on several streams: those that use its workspace run one
behind the other, whatever streams they are on."""
import pytest
import torch

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu
SLEEP = 200_000_000  # cycles: some 0.1 s, much longer than any call here


def _loss(seed):
    """A call whose partial sums of many chunks lie in the workspace, and its results."""
    g = torch.Generator().manual_seed(seed)
    x, w = torch.rand(9000, 4, 32, generator=g).cuda(), torch.rand(4, 32, generator=g).cuda()
    t = (torch.rand(9000, generator=g) < 0.5).float().cuda()
    return lambda tr: tr.loss(x, w, t)


def _draws(seed):
    """Rows cut over many workgroups, whose bins and sums lie in the workspace."""
    g = torch.Generator().manual_seed(seed)
    scores, u = torch.randn(3, 50000, generator=g).cuda(), torch.rand(3, 500, generator=g, dtype=torch.float64).cuda()
    return lambda tr: tr.sample(scores, u, top_k=20000, top_p=0.9)


def _grad(seed):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.rand(9000, 4, 32, generator=g).cuda(), torch.rand(4, 8, 32, generator=g).cuda()
    dy = torch.randn(9000, 4, 8, generator=g).cuda()
    return lambda tr: tr.response_grad(x, w, dy)[:2]


CALLS = [(_loss, _loss), (_draws, _draws), (_grad, _grad), (_loss, _draws), (_draws, _grad)]


@pytest.mark.parametrize("first,second", CALLS)
@pytest.mark.parametrize("captured", [False, True])
def test_calls_on_two_streams_follow_each_other(first, second, captured):
    """The second stream's call waits for the first stream's, which waits for its
    stream's work: had it not, it would end while that still sleeps."""
    tr = sc.Trainer()
    one, two = first(1), second(2)
    want = [[v.clone() for v in call(tr)] for call in (one, two)]  # (the workspace is grown, too)
    [call(tr) for call in (one, two)]
    a, b, c = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    graph, slept, end = torch.cuda.CUDAGraph(), torch.cuda.Event(), torch.cuda.Event()
    with torch.cuda.stream(a):
        torch.cuda._sleep(SLEEP)
        slept.record()
        got_one = one(tr)
    assert not slept.query()
    if captured:
        with torch.cuda.stream(b):
            graph.capture_begin()
            again = one(tr)
            graph.capture_end()
    with torch.cuda.stream(c):
        got_two = two(tr)
        end.record()
    end.synchronize()
    assert slept.query()
    torch.cuda.synchronize()
    for got, exp in zip((got_one, got_two), want):
        assert all(torch.equal(p, q) for p, q in zip(got, exp))
    if captured:
        for _ in range(3):
            graph.replay()
            other = two(tr)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(again, want[0]))
            assert all(torch.equal(p, q) for p, q in zip(other, want[1]))


@pytest.mark.parametrize("first,second", CALLS)
def test_two_trainers_at_once(first, second):
    """Trainers do not share a workspace: their calls overlap and keep their results."""
    t1, t2 = sc.Trainer(), sc.Trainer()
    one, two = first(3), second(4)
    want = [[v.clone() for v in call(t)] for call, t in ((one, t1), (two, t2))]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s1):
            x = one(t1)
        with torch.cuda.stream(s2):
            y = two(t2)
    torch.cuda.synchronize()
    for got, exp in zip((x, y), want):
        assert all(torch.equal(p, q) for p, q in zip(got, exp))
