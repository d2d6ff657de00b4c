"""Models whose embedding or dropout modules are the user's own.  No GPU."""
import numpy as np
import pytest

import minitorch_amd as mt


def _gpt(embedding):
    model = mt.GPT.__new__(mt.GPT)
    mt.module.Module.__init__(model)
    model.block_size, model.tok_emb, model.pos_emb = 8, embedding, embedding
    return model


class Table(mt.module.Module):
    """An embedding module that knows no scale."""


class Tied(mt.Embedding):
    """One that takes its table from elsewhere."""

    def __init__(self, weight):
        mt.module.Module.__init__(self)
        self.weight = weight


class Quiet(mt.Dropout):
    def __init__(self, p):
        mt.module.Module.__init__(self)
        self.p = p


@pytest.mark.parametrize("embedding", [Table(), Tied(None)])
def test_greedy_decoding_takes_tables_without_a_scale(embedding):
    ids = np.array([[1, 2, 3]])
    assert np.array_equal(_gpt(embedding).generate_greedy(ids, 0), ids)


def test_greedy_decoding_still_refuses_scaled_tables():
    table = Table()
    table.scale = 2.0
    with pytest.raises(NotImplementedError):
        _gpt(table).generate_greedy(np.array([[1]]), 0)


def test_subclasses_with_an_init_of_their_own():
    class Weight:
        def __getitem__(self, idx):
            return ("rows", idx.tolist())

    assert Tied(Weight())(np.array([2, 0])) == ("rows", [2, 0])
    assert Quiet(0.5).rng == "host" and Tied(None).scale is None
