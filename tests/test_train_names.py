"""Names the Trainer's calls take (activations, kinds of residual): an unknown one
is a ValueError like every other refusal, and a KeyError."""
import pytest

from surfcascade_amd import train


@pytest.mark.parametrize("names", [train._ACT, train._RES])
@pytest.mark.parametrize("bad", ["tanh", "Row", "", 0, 1.5, (), object()])
def test_unknown_names(names, bad):
    for kind in (ValueError, KeyError):
        with pytest.raises(kind, match="^(activation|residual) must be one of (None, )?'none'"):
            names[bad]


def test_known_names():
    assert [train._ACT[n] for n in ("none", "sigmoid")] == [0, 1]
    assert [train._RES[n] for n in (None, "none", "row", "full")] == [0, 0, 1, 2]


@pytest.mark.gpu
def test_unknown_names_in_calls():
    import torch
    tr = train.Trainer()
    x, w, d = (torch.zeros(*s, device="cuda") for s in ((5, 3, 32), (3, 32), (5, 3)))
    for call in (lambda: tr.response(x, w, activation="tanh"), lambda: tr.response_grad(x, w, d, activation=None),
                 lambda: tr.response_grad(x, w, d, residual="rows"), lambda: tr.response_grad(x, w, d, residual=d)):
        with pytest.raises(ValueError):
            call()
        with pytest.raises(KeyError):
            call()
