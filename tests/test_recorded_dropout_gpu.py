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


@pytest.mark.parametrize("shape", [(2, 3, 5, 7), (1, 4, 24, 24)])
def test_attention_masks_from_the_device_generator(dev, shape):
    from minitorch_amd import F

    B, H, Tq, Tk = shape
    F.set_dropout_seed(12)
    at = 0
    for _ in range(2):
        mask, scale = F.attention_keep_mask((B, H, Tq, Tk), 0.25, "device")
        want = ref.keep((B * H * Tq, Tk), 0.25, 12, at, 1).reshape(B, H, Tq, Tk)
        assert np.array_equal(mask.numpy()[..., :Tk] != 0, want) and scale == np.float32(1 / 0.75)
        at += (want.size + 3) // 4


def test_host_masks_are_refused_in_a_recorded_step(dev):
    import minitorch_amd as mt

    attn = mt.MultiHeadAttention(32, 2, dropout=0.5)
    step = mt.CapturedStep(lambda x: attn(mt.Tensor(x)), warmup=1)
    x = mt.Tensor(np.ones((1, 4, 32), np.float32)).data
    step(x)
    with pytest.raises(RuntimeError, match="dropout_rng"):
        step(x)


class _Numbers:
    """Stands for a recorded graph in eager steps: F.dropout draws from where a replay of
    the graph would."""

    def __init__(self, seed):
        from minitorch_amd.device import zeros

        self.seed, self.subsequence, self.draws, self.base = seed, 2, 0, zeros((1,), "int64").t

    def step(self, i, fn, *args):
        from minitorch_amd import _lib

        self.draws = 0
        if i:
            self.base.copy_(np.array([i * self.each]))
        _lib._GRAPH[0] = self
        try:
            return fn(*args)
        finally:
            _lib._GRAPH[0] = None
            self.each = self.draws


@pytest.mark.parametrize("whole", [True, False])
def test_a_recorded_gpt_with_dropout_is_the_eager_one(dev, whole):
    """GPT(dropout=..., dropout_rng="device") as the constructor makes it, attention's
    masks included, recorded with its loss, gradients and Adam: every replay's loss and
    the weights after them are those of eager steps that draw the same numbers, to the
    bit.  With GPT.loss, and with the logits and their cross entropy."""
    import minitorch_amd as mt
    from minitorch_amd import F
    from minitorch_amd.device import index_array
    from oracle import gpt as G

    rng = np.random.default_rng(3)
    cfg = G.GPTConfig(301, 24, 64, 4, 2)
    P = G.init_params(cfg, rng)
    x, y = rng.integers(0, cfg.vocab, (4, 24)), rng.integers(0, cfg.vocab, (4, 24))
    batches = [(index_array(np.roll(x, i, 0)), index_array(np.roll(y, i, 0))) for i in range(5)]
    runs = []
    for record in (False, True):
        model = mt.GPT(cfg.vocab, cfg.block, cfg.n_embd, cfg.n_head, cfg.n_layer, dropout=0.1, dropout_rng="device")
        model.load_state_dict(P)
        model.train()
        opt = mt.Adam(model.parameters(), lr=3e-4)
        opt.capturable()

        def step(a, b):
            opt.zero_grad()
            loss = model.loss(a, b) if whole else F.cross_entropy(model(a).reshape(-1, cfg.vocab), b.reshape(-1))
            loss.backward()
            opt.step()
            return loss

        F.set_dropout_seed(21)
        run = mt.CapturedStep(step, opt, warmup=1) if record else step
        numbers = _Numbers(21)
        losses = [float(run(*batches[0]))]  # eager either way: the warm-up
        for i, b in enumerate(batches):
            losses.append(float(run(*b) if record else numbers.step(i, step, *b)))
        runs.append((losses, {k: t.data.numpy() for k, t in model._named_state()}))
    assert runs[0][0] == runs[1][0] and len(set(runs[0][0])) == 6
    for name, value in runs[0][1].items():
        assert np.array_equal(value, runs[1][1][name]), name


def test_dropout_changes_what_attention_adds_up(dev):
    """In training the module's output is the attention under the masks that its seed
    draws; in evaluation there are none."""
    import minitorch_amd as mt
    from minitorch_amd import F

    attn = mt.MultiHeadAttention(32, 2, dropout=0.5, dropout_rng="device")
    x = mt.Tensor(np.random.default_rng(1).standard_normal((2, 6, 32)).astype(np.float32))
    outs = []
    for seed in (1, 1, 2):
        F.set_dropout_seed(seed)
        outs.append(attn(x).numpy())
    assert np.array_equal(outs[0], outs[1]) and not np.array_equal(outs[0], outs[2])
    attn.eval()
    assert np.array_equal(attn(x).numpy(), attn(x).numpy())
