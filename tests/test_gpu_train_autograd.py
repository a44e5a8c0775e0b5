"""What the training operators do beside torch's differentiation: they take no
part in it, and no call looks as if it did."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


def _operands(seed=1, n=9, p=3, h=2):
    g = torch.Generator().manual_seed(seed)
    x, w, b = torch.rand(n, p, 32, generator=g), torch.randn(p, h, 32, generator=g), torch.randn(p, h, generator=g)
    return x.cuda(), w.cuda(), b.cuda()


def _calls(tr):
    x, w, b = _operands()
    t, c = torch.zeros(9, device="cuda"), torch.ones(9, device="cuda")
    dy, u = torch.ones(9, 3, 2, device="cuda"), torch.rand(4, dtype=torch.float64, device="cuda")
    row = torch.ones(9, device="cuda")
    return [(x, lambda v: tr.response(v, w, b)), (w, lambda v: tr.response(x, v, b)), (b, lambda v: tr.response(x, w, v)),
            (row, lambda v: tr.response(x, w, b, residual=v)), (dy, lambda v: tr.response(x, w, b, residual=v)),
            (x, lambda v: tr.loss(v, w, t, b)), (w, lambda v: tr.loss(x, v, t, b)), (b, lambda v: tr.loss(x, w, t, v)),
            (t, lambda v: tr.loss(x, w, v, b)), (c, lambda v: tr.loss(x, w, t, b, weight=v)),
            (w, lambda v: tr.response_grad(x, v, dy, b)), (dy, lambda v: tr.response_grad(x, w, v, b)),
            (row, lambda v: tr.sample(v, u))]


def test_forward_tangents_are_refused(tr):
    """A dual operand's tangent would be lost; inside a level, operands without one
    are taken as anywhere."""
    for operand, call in _calls(tr):
        want = call(operand)
        with fwd.dual_level():
            dual = fwd.make_dual(operand, torch.ones_like(operand))
            with pytest.raises(ValueError, match="tangent"):
                call(dual)
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call(dual)
            got = call(fwd.unpack_dual(dual).primal)
        for a, e in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert (a is None and e is None) or torch.equal(a, e)


def test_out_is_an_in_place_write(tr):
    """A buffer that asks for gradients is refused, and what autograd had saved of
    another is known to be gone."""
    x, w, b = _operands()
    want = tr.response(x, w, b)
    leaf = torch.zeros(9, 3, 2, device="cuda", requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="autograd"):
            tr.response(x, w, b, out=out)
        assert not out.any()
    with torch.no_grad():
        assert torch.equal(tr.response(x, w, b, out=leaf), want)
    saved = torch.ones(9, 3, 2, device="cuda")
    a = torch.ones(9, 3, 2, device="cuda", requires_grad=True)
    product = (a * saved).sum()
    tr.response(x, w, b, out=saved)
    with pytest.raises(RuntimeError, match="inplace"):
        product.backward()
    assert a.grad is None
    with fwd.dual_level():
        dual = fwd.make_dual(torch.zeros(9, 3, 2, device="cuda"), torch.ones(9, 3, 2, device="cuda"))
        with pytest.raises(ValueError, match="tangent"):
            tr.response(x, w, b, out=dual)
    with torch.inference_mode():
        out = torch.empty(9, 3, 2, device="cuda")
        assert torch.equal(tr.response(x, w, b, out=out), want)
    # a view's write is its base's
    base = torch.ones(9, 8, device="cuda")
    product = (torch.ones(9, 8, device="cuda", requires_grad=True) * base).sum()
    tr.response(x, w, b, out=base[:, 1:7])
    with pytest.raises(RuntimeError, match="inplace"):
        product.backward()
