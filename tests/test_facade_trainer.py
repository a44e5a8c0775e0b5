"""The C++ facade's Trainer (include/surfcascade.hpp) over the C ABI."""
import math
import os
import subprocess

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def trainer_bin(tmp_path_factory):
    import surfcascade_amd as sc
    lib = sc.library_path()
    out = str(tmp_path_factory.mktemp("trainer") / "trainer_main")
    subprocess.check_call(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-std=c++17", "-O1", "-I",
                           os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "trainer_main.cpp"),
                           "-o", out, "-L", os.path.dirname(lib), "-lsurfcascade",
                           "-Wl,-rpath," + os.path.dirname(lib)])
    return out


def test_refusal_through_the_facade_header(trainer_bin):
    r = subprocess.run([trainer_bin, "refuse"], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.startswith("-1 samples overlap")


@pytest.mark.gpu
def test_draw_and_loss(trainer_bin):
    """Rows 0 and 2 are drawn (row 1 is masked); with zero weights each loss is
    log 2 and each gradient -1/2 for the positive row, 1/2 for the other."""
    r = subprocess.run([trainer_bin], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    lines = r.stdout.splitlines()
    assert lines[0] == "drawn 0 2"
    for v in lines[1].split()[1:]:
        assert abs(float(v) - 2 * math.log(2)) <= 1e-6
    assert lines[2] == "dw -0.5 0 0.5" and lines[3] == "db 0"
