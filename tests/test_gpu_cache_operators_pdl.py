"""The cache operators under programmatic dependent launch (``NIB_B200_PDL=1``, off by default): a chain of
them gives the same bits with it off and on, eagerly and replayed from a CUDA graph
(``tests/_cache_operators_pdl_child.py``). The suffixes of a shared prefix start without waiting for the
kernel before them, whose start says that everything before it has ended; chunk selection is a cluster
launch with the programmatic attribute."""

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


def _run(pdl: bool) -> dict:
    env = dict(os.environ)
    env.pop("NIB_B200_PDL", None)
    if pdl:
        env["NIB_B200_PDL"] = "1"
    r = subprocess.run([sys.executable, str(ROOT / "tests" / "_cache_operators_pdl_child.py")], env=env, cwd=ROOT,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout.strip().splitlines()[-1])


def test_programmatic_dependent_launch_gives_the_same_bits():
    off, on = _run(False), _run(True)
    assert off["finite"] and on["finite"]
    bits = set(off["eager"] + off["graph"] + on["eager"] + on["graph"])
    assert len(bits) == 1, (off, on)
