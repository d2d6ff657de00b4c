"""Recorded steps that draw dropout masks on the device: reproducible from the seed, and
the same as eager steps that draw the same numbers."""
import numpy as np
import pytest

from oracle import vocab as ref

pytestmark = pytest.mark.gpu


def _recorded(n=3):
    """Record a step of one dropout and replay it: the masks."""
    import minitorch_amd as mt
    from minitorch_amd import F

    step = mt.CapturedStep(lambda x: F.dropout(mt.Tensor(x), 0.5), warmup=1)
    x = mt.Tensor(np.ones((4, 100), np.float32)).data
    step(x)
    return [step(x).numpy() != 0 for _ in range(n)], step.graph


def test_a_seed_and_the_recordings_after_it_give_the_same_masks(dev):
    """Whatever was recorded before in the process, and graphs without dropout between."""
    import minitorch_amd as mt
    from minitorch_amd import F

    runs = []
    for turn in range(3):
        F.set_dropout_seed(31)
        if turn:
            plain = mt.CapturedStep(lambda x: F.gelu(mt.Tensor(x)), warmup=1)
            for _ in range(2):
                plain(mt.Tensor(np.ones((2, 3), np.float32)).data)
            assert plain.graph.subsequence is None
        first, graph = _recorded()
        second, other = _recorded()
        assert (graph.subsequence, other.subsequence) == (2, 3)
        runs.append(first + second)
        _recorded(1)
    for masks in runs[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(masks, runs[0]))
    for i in range(3):
        assert np.array_equal(runs[0][i], ref.keep((4, 100), 0.5, 31, 100 * i, 2))
        assert np.array_equal(runs[0][3 + i], ref.keep((4, 100), 0.5, 31, 100 * i, 3))


def test_a_restart_leaves_recorded_graphs_alone(dev):
    import minitorch_amd as mt
    from minitorch_amd import F

    F.set_dropout_seed(8)
    step = mt.CapturedStep(lambda x: F.dropout(mt.Tensor(x), 0.5), warmup=1)
    x = mt.Tensor(np.ones((4, 100), np.float32)).data
    step(x)
    for i in range(4):
        got = step(x).numpy() != 0
        assert np.array_equal(got, ref.keep((4, 100), 0.5, 8, 100 * i, 2))
        F.set_dropout_seed(9)
