"""Training with a large vocabulary through the public functions and models:
F.embedding, F.dropout, F.linear_cross_entropy, Embedding(scale), Dropout(rng),
GPT.loss, eagerly and in recorded steps, against the float64 forms (oracle.vocab,
oracle.gpt)."""
import numpy as np
import pytest
from test_vocab_gpu import B, U, inside, rounded, tokens, xent_bounds

from oracle import vocab as ref

pytestmark = pytest.mark.gpu


def ids_array(a):
    from minitorch_amd import device

    return device.index_array(np.asarray(a))


def test_embedding_and_gradient(dev):
    import minitorch_amd as mt
    from minitorch_amd import F

    rng = np.random.default_rng(0)
    V, C = 300, 40
    w = rng.standard_normal((V, C)).astype(np.float32)
    ids = np.where(rng.random((6, 50)) < 0.2, -1, rng.integers(0, V, (6, 50)))
    g = rng.standard_normal((6, 50, C)).astype(np.float32)
    for idx in (ids, ids_array(ids)):
        table = mt.Tensor(w, requires_grad=True)
        y = F.embedding(table, idx, scale=8.0)
        inside(y.numpy(), ref.lookup(w, ids.ravel(), 8.0).reshape(y.shape), 0)  # a power of two: exact
        (y * mt.Tensor(g)).sum().backward()
        want, size = ref.lookup_grad(ids.ravel(), g.reshape(-1, C), V, 8.0)
        inside(table.grad.numpy(), want, 64 * U * size)
        # a second use of the table adds to its gradient
        first = table.grad.numpy().copy()
        (F.embedding(table, idx, scale=8.0) * mt.Tensor(g)).sum().backward()
        inside(table.grad.numpy(), 2 * first, 4 * U * np.abs(first) + 64 * U * size)
    with pytest.raises(IndexError):
        F.embedding(table, np.array([V]))


def test_embedding_layer_scales(dev):
    import minitorch_amd as mt

    emb = mt.Embedding(11, 6, scale=4.0)
    ids = np.array([[0, 10, -1]])
    assert np.array_equal(emb(ids).numpy(), ref.lookup(emb.weight.numpy(), ids.ravel(), 4.0)[None].astype(np.float32))
    plain = mt.Embedding(11, 6)
    assert np.array_equal(plain(ids[:, :2]).numpy(), plain.weight.numpy()[ids[:, :2]])


@pytest.mark.parametrize("residual", [False, True])
def test_dropout_and_gradient(dev, residual):
    import minitorch_amd as mt
    from minitorch_amd import F

    rng = np.random.default_rng(1)
    x, r, g = (rng.standard_normal((5, 7, 33)).astype(np.float32) for _ in range(3))
    F.set_dropout_seed(77)
    at = 0
    for _ in range(2):  # the second call draws other numbers
        tx, tr = mt.Tensor(x, requires_grad=True), mt.Tensor(r, requires_grad=True)
        y = F.dropout(tx, 0.3, residual=tr if residual else None)
        keep = ref.keep((1, x.size), 0.3, 77, at, subsequence=1).reshape(x.shape)
        scaled = np.where(keep, x * np.float32(1 / 0.7), np.float32(0))
        assert np.array_equal(y.numpy(), r + scaled if residual else scaled)
        (y * mt.Tensor(g)).sum().backward()
        assert np.array_equal(tx.grad.numpy(), np.where(keep, g * np.float32(1 / 0.7), np.float32(0)))
        if residual:
            assert np.array_equal(tr.grad.numpy(), g)
        at += (x.size + 3) // 4


def test_dropout_of_one_tensor_twice(dev):
    """x as input and residual, and a second consumer: gradients add up."""
    import minitorch_amd as mt
    from minitorch_amd import F

    x = np.random.default_rng(2).standard_normal((9, 31)).astype(np.float32)
    F.set_dropout_seed(5)
    t = mt.Tensor(x, requires_grad=True)
    (F.dropout(t, 0.5, residual=t) + t).sum().backward()
    keep = ref.keep((1, x.size), 0.5, 5, 0, subsequence=1).reshape(x.shape)
    assert np.array_equal(t.grad.numpy(), 2 + 2.0 * keep)


def test_dropout_layer(dev):
    import minitorch_amd as mt
    from minitorch_amd import F

    x = mt.Tensor(np.ones((4, 100), np.float32))
    layer = mt.Dropout(0.25, rng="device")
    F.set_dropout_seed(3)
    keep = ref.keep((1, 400), 0.25, 3, 0, subsequence=1).reshape(4, 100)
    assert np.array_equal(layer(x).numpy() != 0, keep)
    layer.eval()
    assert layer(x) is x
    with pytest.raises(ValueError):
        mt.Dropout(0.5, rng="gpu")


def test_dropout_in_a_recorded_step(dev):
    """Every replay draws other numbers, forward and backward alike, whatever runs
    eagerly in between."""
    import minitorch_amd as mt
    from minitorch_amd import F
    from minitorch_amd.device import DeviceArray, zeros

    F.set_dropout_seed(13)
    n, out = 1000, {}

    def step(x):
        t = mt.Tensor(x, requires_grad=True)
        a = F.dropout(t, 0.5)
        b = F.dropout(a, 0.2, residual=a)
        b.sum().backward()
        out.update(b=b, g=t.grad)
        return b

    one = mt.CapturedStep(step, warmup=1)
    x = mt.Tensor(np.ones((10, 100), np.float32)).data
    one(x)
    sub = None
    for i in range(5):
        b = one(x).numpy()
        sub = one.graph.subsequence
        k1 = ref.keep((1, n), 0.5, 13, 500 * i, sub).reshape(10, 100)
        k2 = ref.keep((1, n), 0.2, 13, 500 * i + 250, sub).reshape(10, 100)
        more = np.float32(1) + np.where(k2, np.float32(1.25), np.float32(0))
        assert np.array_equal(b, np.where(k1, np.float32(2) * more, np.float32(0)))
        assert np.array_equal(out["g"].numpy(), np.where(k1, np.float32(2) * more, np.float32(0)))
        F.dropout(mt.Tensor(zeros((3, 5))), 0.5).numpy()  # eager draws move nothing in the graph
        zeros((64,)).numpy()
    assert sub > 1


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tied", [False, True])
def test_linear_cross_entropy(dev, tied, dtype):
    import minitorch_amd as mt
    from minitorch_amd import F
    from minitorch_amd.device import from_host

    rng = np.random.default_rng(6)
    n, C, V = 150, 40, 700
    x = rounded(rng.standard_normal((3, n // 3, C)), dtype)
    w = rounded(rng.standard_normal((C, V)) / 3, dtype)
    b = rng.standard_normal(V).astype(np.float32)
    labels = tokens(rng, n, V)
    labels[labels >= V] = -1
    r = ref.linear_xent(x.reshape(n, C), w, labels, b)
    _, _, bl, bx, bw, bb = xent_bounds(x.reshape(n, C), w, b, r, dtype, "float32")
    for lab in (labels.reshape(3, -1), ids_array(labels)):
        tx = mt.Tensor(from_host(x, dtype), requires_grad=True)
        table = mt.Tensor(from_host(w.T if tied else w, dtype), requires_grad=True)
        tb = mt.Tensor(b, requires_grad=True)
        loss = F.linear_cross_entropy(tx, table.transpose() if tied else table, tb, lab, logits_bytes=64 * V * 4)
        inside(loss.numpy(), r["loss"], bl)
        (loss * 3.0).backward()
        for t, want, bd in ((tx, r["dx"].reshape(x.shape), bx.reshape(x.shape)),
                            (table, r["dw"].T if tied else r["dw"], bw.T if tied else bw), (tb, r["db"], bb)):
            inside(t.grad.numpy(), 3 * want, 3 * bd + 4 * U * np.abs(want))
        first = [t.grad.numpy().copy() for t in (tx, table, tb)]
        # once more into the same gradients
        (F.linear_cross_entropy(tx, table.transpose() if tied else table, tb, lab) * 3.0).backward()
        for t, f, bd in zip((tx, table, tb), first, (bx.reshape(x.shape), bw.T if tied else bw, bb)):
            inside(t.grad.numpy(), 2 * f, 6 * bd + 8 * U * np.abs(f))
    with mt.no_grad():
        inside(F.linear_cross_entropy(tx, table.transpose() if tied else table, tb, labels).numpy(), r["loss"], bl)
    with pytest.raises(IndexError):
        F.linear_cross_entropy(tx, table.transpose() if tied else table, tb, np.full(n, V))
    with pytest.raises(ValueError):
        F.linear_cross_entropy(tx, table.transpose() if tied else table, tb, labels[:-1])


def test_linear_cross_entropy_frozen(dev):
    import minitorch_amd as mt
    from minitorch_amd import F

    rng = np.random.default_rng(7)
    x, w = rng.standard_normal((20, 8)).astype(np.float32), rng.standard_normal((8, 30)).astype(np.float32)
    labels = rng.integers(0, 30, 20)
    r = ref.linear_xent(x, w, labels)
    tx, tw = mt.Tensor(x), mt.Tensor(w, requires_grad=True)
    F.linear_cross_entropy(tx, tw, None, labels).backward()
    inside(tw.grad.numpy(), r["dw"], xent_bounds(x, w, None, r, "float32", "float32")[4])
    assert tx.grad is None


def _gpt(dropout=0.0, rng="host"):
    import minitorch_amd as mt
    from oracle import gpt as G

    cfg = G.GPTConfig(301, 24, 64, 4, 2)
    P = G.init_params(cfg, np.random.default_rng(8))
    model = mt.GPT(cfg.vocab, cfg.block, cfg.n_embd, cfg.n_head, cfg.n_layer, dropout=dropout, dropout_rng=rng)
    model.load_state_dict(P)
    return model, cfg, P


def test_gpt_loss_matches_the_reference_path(dev):
    """GPT.loss against the oracle's loss and gradients, at the bounds of the fp32
    path (test_gpt_gpu): loss 1e-5 relative, entries 1e-3 of their tensor's largest."""
    from oracle import gpt as G

    model, cfg, P = _gpt()
    rng = np.random.default_rng(9)
    x, y = rng.integers(0, cfg.vocab, (5, cfg.block)), rng.integers(0, cfg.vocab, (5, cfg.block))
    want, _, grads = G.gpt_loss_and_grads(P, x, y, cfg)
    loss = model.loss(x, y)
    assert abs(float(loss) - want) <= 1e-5 * want
    loss.backward()
    grads = {k: g.g if hasattr(g, "g") else g for k, g in grads.items()}
    for (name, t) in model._named_state():
        # a key bias b adds q.b to all of a row's scores, which its softmax does not
        # see: that gradient is 0, and what stands there is rounding of values as
        # large as the key weights' gradient
        size = np.abs(grads[name.replace("k_proj.bias", "k_proj.weight")]).max()
        assert np.abs(t.grad.numpy() - grads[name]).max() <= 1e-3 * size, name


def test_gpt_loss_of_padded_batches(dev):
    """Padded targets count nowhere: the loss of a padded batch is that of its
    sequences, each with its own tokens, weighted by them."""
    model, cfg, _ = _gpt()
    rng = np.random.default_rng(10)
    x, y = rng.integers(0, cfg.vocab, (3, cfg.block)), rng.integers(0, cfg.vocab, (3, cfg.block))
    lens = [24, 9, 1]
    px, py = x.copy(), y.copy()
    total = 0.0
    for i, n in enumerate(lens):
        px[i, n:] = py[i, n:] = -1
        total += n * float(model.loss(x[i:i + 1, :n], y[i:i + 1, :n]))
    # losses of about 6, each off by some tens of roundings on either side
    assert abs(float(model.loss(px, py)) - total / sum(lens)) <= 200 * U * 6


def test_gpt_training_step_with_device_dropout(dev):
    """Lookup, dropout, blocks, loss, gradients, Adam, recorded and replayed: the
    masks differ from step to step, the losses are those of eager steps that draw
    the same numbers."""
    import minitorch_amd as mt
    from minitorch_amd import F

    rng = np.random.default_rng(11)
    x, y = (rng.integers(0, 301, (4, 24)) for _ in range(2))
    losses = []
    for record in (False, True):
        model, cfg, P = _gpt(0.1, "device")
        for block in model.blocks:
            block.attn.attn_drop.p = 0.0  # its masks are drawn outside recorded steps
        model.train()
        F.set_dropout_seed(21)
        opt = mt.Adam(model.parameters(), lr=3e-4)
        opt.capturable()

        def step(a, b):
            opt.zero_grad()
            loss = model.loss(a, b)
            loss.backward()
            opt.step()
            return loss

        run = mt.CapturedStep(step, opt, warmup=1) if record else step
        dx, dy = ids_array(x), ids_array(y)
        got = [float(run(dx, dy)) for _ in range(6)]
        assert len(set(got)) == 6
        losses.append(got)
    assert losses[0][0] == losses[1][0]  # the eager warm-up step
    assert np.isfinite(losses).all()


def test_greedy_decoding_refuses_scaled_tables(dev):
    import minitorch_amd as mt

    model, cfg, _ = _gpt()
    model.tok_emb = mt.Embedding(cfg.vocab, cfg.n_embd, scale=8.0)
    with pytest.raises(NotImplementedError):
        model.generate_greedy(np.zeros((1, 4), np.int64), 3)


@pytest.mark.parametrize("first", [0, 1])
def test_a_transposed_table_with_two_uses(dev, first):
    """Its gradient arrives in the table's layout from one use and row by row from
    the other, in either order."""
    import minitorch_amd as mt
    from minitorch_amd import F

    rng = np.random.default_rng(12)
    table = mt.Tensor(rng.standard_normal((30, 8)).astype(np.float32), requires_grad=True)
    x = mt.Tensor(rng.standard_normal((20, 8)).astype(np.float32), requires_grad=True)
    labels = rng.integers(0, 30, 20)
    F.set_dropout_seed(4)
    w = table.transpose()
    uses = [lambda: F.linear_cross_entropy(x, w, None, labels), lambda: F.dropout(w, 0.5).sum()]
    a, b = uses[first](), uses[1 - first]()
    (a + b).backward()
    keep = ref.keep((1, 240), 0.5, 4, 0, subsequence=1).reshape(8, 30)
    r = ref.linear_xent(x.numpy(), table.numpy().T, labels)
    bound = xent_bounds(x.numpy(), table.numpy().T, None, r, "float32", "float32")[4].T
    want = (r["dw"] + 2.0 * keep).T
    inside(table.grad.numpy(), want, bound + 2 * U * (np.abs(want) + bound))


def test_shapes_at_the_ends(dev):
    """No rows, one row without a batch axis, 0-d values, transposed inputs."""
    import minitorch_amd as mt
    from minitorch_amd import F

    rng = np.random.default_rng(13)
    w = mt.Tensor(rng.standard_normal((8, 30)).astype(np.float32), requires_grad=True)
    x = mt.Tensor(np.zeros((0, 8), np.float32), requires_grad=True)
    loss = F.linear_cross_entropy(x, w, None, np.zeros(0, np.int64))
    loss.backward()
    assert float(loss) == 0 and not w.grad.numpy().any() and x.grad.numpy().shape == (0, 8)
    assert F.embedding(w, np.zeros((0,), np.int64)).shape == (0, 30)
    assert F.dropout(mt.Tensor(np.zeros((0, 3), np.float32)), 0.5).shape == (0, 3)
    one = rng.standard_normal(8).astype(np.float32)
    t = mt.Tensor(one, requires_grad=True)
    F.linear_cross_entropy(t, w, None, np.array([3])).backward()
    r = ref.linear_xent(one[None], w.numpy(), np.array([3]))
    inside(t.grad.numpy(), r["dx"][0], xent_bounds(one[None], w.numpy(), None, r, "float32", "float32")[3][0])
    w.grad = None
    y = F.embedding(w, np.array(2), scale=2.0)
    y.sum().backward()
    assert np.array_equal(y.numpy().ravel(), 2 * w.numpy()[2])
    assert np.array_equal(w.grad.numpy(), np.where(np.arange(8)[:, None] == 2, 2.0, 0.0) * np.ones(30))
    s = mt.Tensor(np.float32(3), requires_grad=True)
    F.set_dropout_seed(1)
    F.dropout(s, 0.5).backward()
    assert s.grad.numpy().item() in (0.0, 2.0)
    xt = rng.standard_normal((8, 20)).astype(np.float32)
    labels = rng.integers(0, 30, 20)
    tx = mt.Tensor(xt, requires_grad=True)
    F.linear_cross_entropy(tx.transpose(), w, None, labels).backward()
    r = ref.linear_xent(xt.T, w.numpy(), labels)
    inside(tx.grad.numpy(), r["dx"].T, xent_bounds(xt.T, w.numpy(), None, r, "float32", "float32")[3].T)
