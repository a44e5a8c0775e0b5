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
