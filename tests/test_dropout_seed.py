"""The seed of F.dropout's generator where nobody sets one.  No GPU."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from minitorch_amd import functional as F

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture
def fresh(monkeypatch):
    """The generator as in a process that has not used it, and NumPy's state kept."""
    state = np.random.get_state()
    monkeypatch.setattr(F, "_LAYER_RNG", {"seed": None, "offset": 0, "graphs": 0})
    yield F._LAYER_RNG
    np.random.set_state(state)


def test_the_seed_comes_from_numpy_s(fresh):
    seeds = []
    for s in (1, 2, 1):
        fresh.update(seed=None, offset=0)
        np.random.seed(s)
        a, b = F._draw(10), F._draw(3)
        assert a["seed"] == b["seed"] and (a["offset"], b["offset"]) == (0, 10)
        seeds.append(a["seed"])
    assert seeds[0] == seeds[2] != seeds[1] and 0 <= min(seeds) and max(seeds) < 1 << 63


def test_a_seed_that_was_set_takes_nothing_from_numpy(fresh):
    np.random.seed(5)
    before = np.random.get_state()[1:3]
    F.set_dropout_seed(0)
    assert F._draw(4) == dict(seed=0, offset=0, subsequence=1)
    after = np.random.get_state()[1:3]
    assert np.array_equal(before[0], after[0]) and before[1] == after[1]


def test_processes_draw_different_masks():
    code = "from minitorch_amd import functional as F; print(F._draw(1)['seed'])"
    out = [subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, check=True).stdout for _ in range(2)]
    assert out[0] != out[1]
