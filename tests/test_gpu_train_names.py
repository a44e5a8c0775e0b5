"""Unknown names in the Trainer's calls, which are refused before anything runs."""
import pytest

from surfcascade_amd import train


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
