"""The paged cache as the framework uses it: PagedKVCache's pages, generation
through it against generation without, and training on token_logprobs, eagerly
and as a recorded step.

Tokens drawn with one seed have to be the same whatever cache holds the keys:
the logits differ by fp32 rounding only (some 1e-6 of their size), far less than
what moves a draw.  Log probabilities are compared at 1e-4: the logits' own
1e-5 of values up to 8, as the bars of the GPT tests have it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def model(seed=0, block=64, n_embd=64, n_head=2, n_layer=2, vocab=50):
    import minitorch_amd as mt

    m = mt.GPT(vocab, block, n_embd=n_embd, n_head=n_head, n_layer=n_layer)
    # larger than at the start of training, so that attention is not uniform
    return m.init_weights(np.random.default_rng(seed), std=0.15)


def logprobs_of(m, ids, T0, temperature):
    """log softmax of the model's full-context logits at the tokens after T0."""
    import minitorch_amd as mt

    with mt.no_grad():
        x = m(ids).data.numpy().astype(np.float64)[:, T0 - 1:-1] / temperature
    x = x - x.max(-1, keepdims=True)
    x = x - np.log(np.exp(x).sum(-1, keepdims=True))
    return np.take_along_axis(x, ids[:, T0:, None], -1)[..., 0]


@pytest.mark.parametrize("page,T0", [(16, 20), (5, 20), (16, 1)])
def test_generate_through_pages(dev, page, T0):
    m = model()
    rng = np.random.default_rng(1)
    idx = rng.integers(0, 50, (3, T0))
    np.random.seed(5)
    want = m.generate(idx, 30, temperature=0.8)
    np.random.seed(5)
    cache = m.paged_cache(3, page=page)
    got, lp = m.generate(idx, 30, temperature=0.8, cache=cache, return_logprobs=True)
    assert np.array_equal(got, want)
    assert np.abs(lp - logprobs_of(m, got, T0, 0.8)).max() <= 1e-4
    assert [cache.length(b) for b in range(3)] == [T0 + 29] * 3
    used = 3 * -(-(T0 + 29) // page)
    assert cache.free_pages == cache.n_pages - used
    for b in range(3):
        cache.release(b)
    assert cache.free_pages == cache.n_pages
    np.random.seed(5)  # and again, in the pages given back
    assert np.array_equal(m.generate(idx, 30, temperature=0.8, cache=cache), want)


def test_generate_logprobs_without_a_cache(dev):
    m = model()
    idx = np.random.default_rng(2).integers(0, 50, (2, 7))
    np.random.seed(3)
    got, lp = m.generate(idx, 9, return_logprobs=True)
    np.random.seed(3)
    assert np.array_equal(got, m.generate(idx, 9))
    assert np.abs(lp - logprobs_of(m, got, 7, 1.0)).max() <= 1e-4
    ids, none = m.generate(idx, 0, return_logprobs=True)
    assert np.array_equal(ids, idx) and none.shape == (2, 0)


def test_generate_with_bf16_pages(dev):
    """Keys and values rounded to bf16 (half a step 2^-8 each): logits of
    values up to 8 move by some 2^-8 of that, through two layers."""
    m = model()
    idx = np.random.default_rng(4).integers(0, 50, (2, 12))
    np.random.seed(6)
    got, lp = m.generate(idx, 20, cache=m.paged_cache(2, dtype="bfloat16"), return_logprobs=True)
    assert np.abs(lp - logprobs_of(m, got, 12, 1.0)).max() <= 16 * 8 * 2.0 ** -8


def test_bounded_cache_that_never_fills_changes_nothing(dev):
    m = model()
    idx = np.random.default_rng(7).integers(0, 50, (2, 10))
    np.random.seed(8)
    want = m.generate(idx, 20)
    np.random.seed(8)
    cache = m.paged_cache(2, max_tokens=48, keep=30, slack=10, page=8)
    assert np.array_equal(m.generate(idx, 20, cache=cache), want)


def test_bounded_cache_stays_bounded(dev):
    m = model()
    idx = np.random.default_rng(9).integers(0, 50, (2, 25))
    cache = m.paged_cache(2, max_tokens=32, keep=16, recent=4, slack=5, page=8)
    np.random.seed(1)
    first, lp = m.generate(idx, 35, cache=cache, return_logprobs=True)
    assert np.isfinite(lp).all() and (lp <= 0).all()
    assert all(16 <= cache.length(b) <= 21 for b in range(2))
    assert cache.free_pages == cache.n_pages - sum(-(-cache.length(b) // 8) for b in range(2))
    assert np.array_equal(cache.lengths.numpy(), [cache.length(b) for b in range(2)])
    for b in range(2):
        cache.release(b)
    np.random.seed(1)
    again = m.generate(idx, 35, cache=cache)
    assert np.array_equal(again, first)


def test_trim_keeps_what_was_attended_and_the_latest(dev):
    """After a prompt and one cut, each head's rows are the prompt's, in order,
    the last `recent` among them and the others those of greatest weight."""
    import minitorch_amd as mt
    from minitorch_amd import device

    m = model(n_layer=1)
    T0, keep, recent = 30, 12, 3
    idx = np.random.default_rng(11).integers(0, 50, (2, T0))
    full = m.paged_cache(2, page=8, keep=40, slack=4, max_tokens=60, observe=5)
    cut = m.paged_cache(2, page=8, keep=keep, recent=recent, slack=0, max_tokens=32, observe=5)
    pos = m._positions(64)
    with mt.no_grad():
        x = m.tok_emb(idx) + m.pos_emb(device.DeviceArray(pos.t[:T0]))
        for c in (full, cut):
            c.reserve(T0)
            m.blocks[0].forward_paged(x, c, 0)
    w = cut.weights[0].numpy().copy()
    assert np.array_equal(w[..., :T0], full.weights[0].numpy()[..., :T0])
    # five positions observed, each with weight 1 a head
    assert np.abs(w.sum(-1) - 5).max() < 1e-5
    assert not full.trim() and cut.trim()
    rows = lambda c, n: [c.k[0].numpy()[c._tab[b]].transpose(1, 0, 2, 3).reshape(2, -1, 32)[:, :n] for b in range(2)]
    for b, (all_rows, kept) in enumerate(zip(rows(full, T0), rows(cut, keep))):
        for h in range(2):
            old = np.sort(np.argsort(-w[b, h, :T0 - recent], kind="stable")[:keep - recent])
            want = np.concatenate([old, np.arange(T0 - recent, T0)])
            assert np.array_equal(kept[h], all_rows[h][want])
            assert np.array_equal(cut.weights[0].numpy()[b, h, :keep], w[b, h, want])


def test_cache_refusals(dev):
    import minitorch_amd as mt

    for bad in (dict(page=0), dict(dtype="int32"), dict(keep=0), dict(keep=8, recent=9), dict(keep=63, slack=4),
                dict(recent=3), dict(pages=0)):
        with pytest.raises(ValueError):
            mt.PagedKVCache(1, 2, 32, 2, 64, **bad)
    with pytest.raises(ValueError, match="head_dim"):
        mt.PagedKVCache(1, 2, 48, 2, 64)
    c = mt.PagedKVCache(1, 2, 32, 2, 64, page=8, pages=5)
    for n in (0, -1, [1, -1]):
        with pytest.raises(ValueError):
            c.reserve(n)
    with pytest.raises(ValueError, match="exceed"):
        c.reserve([65, 1])
    with pytest.raises(RuntimeError, match="pages"):
        c.reserve([33, 8])
    assert c.free_pages == 5 and c.length(0) == 0  # nothing changed
    c.reserve([32, 8])
    assert c.free_pages == 0
    m = model()
    idx = np.zeros((2, 10), np.int64)
    with pytest.raises(ValueError, match="batch"):
        m.generate(idx, 3, cache=m.paged_cache(3))
    with pytest.raises(ValueError, match="block_size"):
        m.generate(idx, 60, cache=m.paged_cache(2))
    used = m.paged_cache(2)
    m.generate(idx, 3, cache=used)
    with pytest.raises(ValueError, match="empty"):
        m.generate(idx, 3, cache=used)


def test_sequences_that_get_no_row_are_left_as_they_are(dev):
    """A step of some sequences: the others' rows, weights and lengths stay, and
    their queries see nothing."""
    import minitorch_amd as mt
    from minitorch_amd import device

    rng = np.random.default_rng(21)
    c = mt.PagedKVCache(1, 2, 32, 3, 64, page=8, keep=40, slack=4)

    def rows(T):
        return device.from_host(rng.standard_normal((3, 2, T, 32)), np.float32).t

    c.reserve([3, 12, 0])
    c.append(0, rows(12), rows(12))
    first = c.attend(0, rows(1), 0.2).numpy()  # of the prompts: counts weights
    assert np.abs(first[:2]).min() > 0 and not first[2].any()
    weights = c.weights[0].numpy()
    before = [p.numpy().view(np.uint32) for p in (c.k[0], c.v[0])]
    c.reserve([1, 0, 1])
    c.append(0, rows(1), rows(1))
    out = c.attend(0, rows(1), 0.2).numpy()
    assert not out[1].any() and np.abs(out[[0, 2]]).min() > 0
    now = c.weights[0].numpy()
    assert np.array_equal(now[1], weights[1]) and np.array_equal(c.lengths.numpy(), [4, 12, 1])
    assert np.abs(now.sum((1, 2)) - weights.sum((1, 2)) - [2, 0, 2]).max() < 1e-5
    for p, was in zip((c.k[0], c.v[0]), before):
        assert (p.numpy().view(np.uint32) != was).any((2, 3)).sum() == 4  # a page and head each of two sequences
    c.reserve(1)  # and all again
    c.append(0, rows(1), rows(1))
    assert np.abs(c.attend(0, rows(1), 0.2).numpy()).min() > 0


def test_append_refuses_other_rows_than_reserved(dev):
    import minitorch_amd as mt

    c = mt.PagedKVCache(1, 2, 32, 2, 64, page=8)
    k = mt.Tensor(np.zeros((2, 2, 3, 32), np.float32)).data.t
    c.reserve([2, 1])
    with pytest.raises(ValueError, match="reserved"):
        c.append(0, k, k)
    m = model(n_layer=1)
    bounded = m.paged_cache(2, max_tokens=40, keep=20)
    bounded.reserve([5, 4])
    with mt.no_grad(), pytest.raises(ValueError, match="one length"):
        m.blocks[0].forward_paged(mt.Tensor(np.zeros((2, 5, 64), np.float32)), bounded, 0)
    c = m.paged_cache(2)
    for _ in range(2):
        c.reserve(3)
    with mt.no_grad(), pytest.raises(ValueError, match="empty sequences"):
        m.blocks[0].forward_paged(mt.Tensor(np.zeros((2, 3, 64), np.float32)), c, 0)


# ---------------------------------------------------------------------------
# training on log probabilities
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("N,V", [(7, 33), (40, 1500)])
def test_token_logprobs_is_cross_entropys_negative(dev, N, V):
    """mean(-logprob) and its gradient are cross_entropy's."""
    import minitorch_amd as mt

    rng = np.random.default_rng(V)
    x = rng.standard_normal((N, V)).astype(np.float32) * 3
    tok = rng.integers(0, V, N)
    a, b = mt.Tensor(x, requires_grad=True), mt.Tensor(x, requires_grad=True)
    lp, ent, ids, tops = mt.F.token_logprobs(a, tok, top=3)
    loss = (-lp).mean()
    loss.backward()
    want = mt.F.cross_entropy(b, tok)
    want.backward()
    assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(want))
    # a probability to 1e-4 relative, over N rows
    g, w = a.grad.numpy(), b.grad.numpy()
    assert np.all(np.abs(g - w) <= 1e-4 * np.abs(w) + 1e-9)
    assert ids.shape == (N, 3) and np.array_equal(ids.numpy()[:, 0], x.argmax(1))


def test_token_logprobs_gradients_add_up(dev):
    """A loss of both outputs, twice, with a temperature and rows without a
    token, against the float64 form; the logits' other consumer adds to it."""
    import minitorch_amd as mt
    from oracle import paged as ref

    rng = np.random.default_rng(3)
    N, V, temperature = 9, 70, 0.5
    x = rng.standard_normal((N, V)).astype(np.float32)
    tok = rng.integers(0, V, N)
    tok[[2, 5]] = -1
    adv = rng.standard_normal(N).astype(np.float32)
    t = mt.Tensor(x, requires_grad=True)
    lp, ent, _, _ = mt.F.token_logprobs(t, tok, temperature=temperature)
    ((lp * mt.Tensor(adv)).sum() + ent.sum() * 0.25 + t.sum()).backward()
    want = ref.logprobs_grad(x, tok, adv, np.full(N, 0.25, np.float32), 2.0) + 1
    got = t.grad.numpy()
    assert np.all(np.abs(got - want) <= 1e-5 * (1 + np.abs(want)))
    assert np.all(lp.numpy()[[2, 5]] == 0)
    # the entropy alone
    t = mt.Tensor(x, requires_grad=True)
    mt.F.token_logprobs(t, tok)[1].sum().backward()
    want = ref.logprobs_grad(x, tok, np.zeros(N, np.float32), np.ones(N, np.float32))
    assert np.all(np.abs(t.grad.numpy() - want) <= 1e-5)
    with mt.no_grad():
        lp, _, _, _ = mt.F.token_logprobs(t, tok)
    assert not lp.requires_grad


def test_token_logprobs_refusals(dev):
    import minitorch_amd as mt

    x = mt.Tensor(np.zeros((3, 5), np.float32))
    with pytest.raises(IndexError):
        mt.F.token_logprobs(x, [0, 1, 5])
    with pytest.raises(ValueError, match="one token"):
        mt.F.token_logprobs(x, [0, 1])
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            mt.F.token_logprobs(x, [0, 1, 2], temperature=bad)
    for bad in (-1, 6, 65):
        with pytest.raises(ValueError, match="top"):
            mt.F.token_logprobs(x, [0, 1, 2], top=bad)


def test_recorded_training_step_on_logprobs(dev):
    """A policy-gradient step (advantage times log probability, an entropy
    bonus) recorded and replayed, with an eager graph of the same parameters
    alive: the eager steps' losses and parameters, bit for bit."""
    import minitorch_amd as mt
    from minitorch_amd import device

    rng = np.random.default_rng(13)
    B, T, V = 4, 16, 50
    data = [(rng.integers(0, V, (B, T)), rng.integers(0, V, B * T)) for _ in range(7)]
    adv = rng.standard_normal(B * T).astype(np.float32)

    def run(captured):
        m = model(seed=2)
        opt = mt.Adam(m.parameters(), lr=1e-3).capturable()
        weight = mt.Tensor(adv)

        def step(i, y):
            opt.zero_grad()
            logits = m(i).reshape(-1, V)
            lp, ent, _, _ = mt.F.token_logprobs(logits, y)
            loss = -(lp * weight).mean() - ent.mean() * 0.01
            loss.backward()
            opt.step()
            return loss

        rec = mt.CapturedStep(step, optimizer=opt) if captured else step
        losses = []
        for i, y in data:
            keep = mt.F.token_logprobs(m(i).reshape(-1, V), y)[0].sum()  # lives over the step
            losses.append(rec(device.index_array(i), device.index_array(y)).numpy().item())
            assert np.isfinite(float(keep))
        return losses, [p.data.numpy() for p in m.parameters()]

    eager, recorded = run(False), run(True)
    assert eager[0] == recorded[0]
    assert all(np.array_equal(a, b) for a, b in zip(eager[1], recorded[1]))


# ---------------------------------------------------------------------------
# steps that are refused or fail, and pools that are just large enough
# ---------------------------------------------------------------------------


def run_paged(m, cache, tokens, first):
    """Logits (B, T, V) of tokens (B, T) at positions first[b] on, whose rows
    the cache has reserved."""
    import minitorch_amd as mt
    from minitorch_amd import device

    tokens = np.asarray(tokens)
    pos = np.asarray(first)[:, None] + np.arange(tokens.shape[1])
    with mt.no_grad():
        x = m.tok_emb(device.index_array(tokens)) + m.pos_emb(device.index_array(pos))
        for i, block in enumerate(m.blocks):
            x = block.forward_paged(x, cache, i)
        return m.lm_head(m.ln_f(x)).data.numpy()


def state(c):
    """What a cache holds, as far as its calls can tell."""
    return dict(lengths=c.lengths.numpy().tolist(), host=[c.length(b) for b in range(c.batch)],
                table=c.table.numpy().tolist(), pages=c._tab.tolist(), free=sorted(c._free))


@pytest.mark.parametrize("keep", [None, 20])
def test_rows_of_a_refused_step_are_taken_back(dev, keep):
    """A step that is refused after its rows were reserved leaves the cache as
    it was before; the next step's logits are those of a cache that never saw it,
    bit for bit."""
    import minitorch_amd as mt

    m = model()
    rng = np.random.default_rng(31)
    prompt, step = rng.integers(0, 50, (2, 7)), rng.integers(0, 50, (2, 1))
    caches = [m.paged_cache(2, page=4, max_tokens=40, keep=keep) for _ in range(2)]
    for c in caches:
        c.reserve(7)
        run_paged(m, c, prompt, [0, 0])
    c = caches[0]
    before = state(c)

    def refused(n, T, match):
        c.reserve(n)
        assert state(c) != before
        with pytest.raises(ValueError, match=match):
            run_paged(m, c, rng.integers(0, 50, (2, T)), [7, 7])
        assert state(c) == before

    refused(3, 3, "empty sequences")
    refused([2, 0], 2, "empty sequences")
    refused(1, 3, "one new token|reserved")
    refused([1, 3], 1, "reserved")
    c.reserve([0, 6])  # rows of a wrong head size, refused by the kernel's wrapper
    k = mt.Tensor(np.zeros((2, 2, 6, 16), np.float32)).data.t
    with pytest.raises(ValueError):
        c.append(0, k, k)
    assert state(c) == before
    c.reserve([5, 1])
    c.undo()
    c.undo()  # there is nothing more to take back
    assert state(c) == before
    out = []
    for c in caches:
        c.reserve(1)
        out.append(run_paged(m, c, step, [7, 7]))
    assert np.array_equal(*out) and np.isfinite(out[0]).all()
    if keep:
        for i in range(2):
            assert np.array_equal(caches[0].weights[i].numpy(), caches[1].weights[i].numpy())
    # a call that reserved nothing takes nothing of the step before it
    before = state(c)
    for T in (2, 3):
        with pytest.raises(ValueError, match="one new token"):
            run_paged(m, c, rng.integers(0, 50, (2, T)), [8, 8])
    with pytest.raises(ValueError, match="reserved"):
        c.append(1, k, k)
    assert state(c) == before and c.length(0) == 8


def test_a_refused_prompt_leaves_an_empty_cache(dev):
    m = model()
    c = m.paged_cache(2, max_tokens=40, keep=20)
    before = state(c)
    c.reserve([5, 4])
    with pytest.raises(ValueError, match="one length"):
        run_paged(m, c, np.zeros((2, 5), np.int64), [0, 0])
    assert state(c) == before
    idx = np.random.default_rng(32).integers(0, 50, (2, 6))
    np.random.seed(2)
    want = m.generate(idx, 8)
    np.random.seed(2)
    assert np.array_equal(m.generate(idx, 8, cache=c), want)


def test_undo_clears_the_rows_weights(dev):
    """Weights that a step counted for rows that are then taken back."""
    import minitorch_amd as mt
    from minitorch_amd import device

    rng = np.random.default_rng(33)
    rows = lambda T: device.from_host(rng.standard_normal((2, 2, T, 32)), np.float32).t
    c = mt.PagedKVCache(2, 2, 32, 2, 64, page=8, keep=40, slack=4)
    c.reserve([3, 12])
    for i in range(2):
        c.append(i, rows(12), rows(12))
        c.attend(i, rows(1), 0.2)
    c.reserve([2, 1])
    for i in range(2):
        c.append(i, rows(2), rows(2))
        c.attend(i, rows(1), 0.2)
        assert (c.weights[i].numpy()[0, :, 3:5] > 0).all() and (c.weights[i].numpy()[1, :, 12] > 0).all()
    c.undo()
    assert [c.length(b) for b in range(2)] == [3, 12]
    for i in range(2):
        w = c.weights[i].numpy()
        assert not w[0, :, 3:].any() and not w[1, :, 12:].any()
        assert (w[0, :, :3] > 0).all() and (w[1, :, :12] > 0).all()
    c.reserve(1)
    c.release(0)  # gives its row back by itself
    c.undo()
    assert [c.length(b) for b in range(2)] == [0, 12] and c.lengths.numpy().tolist() == [0, 12]
    assert sorted(c._free + [i for i in c._tab.ravel() if i >= 0]) == list(range(c.n_pages))


def test_a_generation_that_fails_leaves_written_rows_alone(dev, monkeypatch):
    """A failure in a layer of the fourth step: its rows are taken back."""
    m = model()
    c = m.paged_cache(2, page=4)
    idx = np.random.default_rng(44).integers(0, 50, (2, 6))
    work, calls = m.blocks[1].forward_paged, []

    def fails(x, cache, layer):
        calls.append(1)
        if len(calls) == 4:
            raise MemoryError("planted")
        return work(x, cache, layer)

    monkeypatch.setattr(m.blocks[1], "forward_paged", fails)
    with pytest.raises(MemoryError):
        m.generate(idx, 10, cache=c)
    assert [c.length(b) for b in range(2)] == [8, 8] and c.lengths.numpy().tolist() == [8, 8]
    assert c.free_pages == c.n_pages - 4


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 62, 2 ** 63 - 1])
def test_reserve_refuses_more_rows_than_an_int_holds(dev, n):
    import minitorch_amd as mt

    c = mt.PagedKVCache(1, 2, 32, 2, 64, page=8)
    c.reserve([3, 5])
    before = state(c)
    for rows in (n, [n, 1], [1, n], np.array([n, n])):
        with pytest.raises(ValueError, match="exceed"):
            c.reserve(rows)
        assert state(c) == before


@pytest.mark.parametrize("keep", [None, 30])
def test_prompt_into_a_released_slot(dev, keep):
    """A sequence that ended gives its slot to a new prompt while the others
    hold theirs: its logits, and theirs from then on, against the whole model's
    over each sequence."""
    m = model()
    rng = np.random.default_rng(34)
    c = m.paged_cache(3, page=4, max_tokens=48, keep=keep, observe=4)
    held = [list(rng.integers(0, 50, 9)) for _ in range(3)]
    c.reserve(9)
    run_paged(m, c, held, [0, 0, 0])

    def steps(n):
        for _ in range(n):
            new = rng.integers(0, 50, (3, 1))
            at = [len(x) for x in held]
            for x, t in zip(held, new[:, 0]):
                x.append(t)
            c.reserve(1)
            got = run_paged(m, c, new, at)
            for b, x in enumerate(held):
                want = m(np.array([x])).data.numpy()[0, -1]
                assert np.abs(got[b, 0] - want).max() <= 1e-4, b

    steps(2)
    c.release(1)
    held[1] = list(rng.integers(0, 50, 6))
    if keep:
        weights = [w.numpy() for w in c.weights]
    c.reserve([0, 6, 0])
    tokens = rng.integers(0, 50, (3, 6))  # the others' rows are nobody's
    tokens[1] = held[1]
    got = run_paged(m, c, tokens, [0, 0, 0])[1]
    assert np.abs(got - m(np.array([held[1]])).data.numpy()[0]).max() <= 1e-4
    assert [c.length(b) for b in range(3)] == [11, 6, 11]
    if keep:  # four positions observed, of weight 1 a head each
        for w, was in zip((w.numpy() for w in c.weights), weights):
            assert np.array_equal(w[[0, 2]], was[[0, 2]])
            assert np.abs(w[1].sum(-1) - 4).max() < 1e-5 and not w[1, :, 6:].any()
    steps(3)
    # a slot's first rows beside another's further ones are no prompt
    c.release(1)
    before = state(c)
    c.reserve([1, 3, 1])
    with pytest.raises(ValueError, match="empty sequences"):
        run_paged(m, c, np.zeros((3, 3), np.int64), [0, 0, 0])
    assert state(c) == before


class Shadow:
    """What a PagedKVCache should hold, in host arrays: each layer and
    sequence's rows (heads, n, D) of keys, values and their weights."""

    def __init__(self, c, rng):
        self.c, self.rng = c, rng
        empty = lambda: np.zeros((c.n_head, 0, c.head_dim), np.float32)
        self.k, self.v = ([[empty() for _ in range(c.batch)] for _ in range(c.n_layer)] for _ in range(2))

    def step(self, n, H):
        """Reserve, append and attend once in every layer; the attention and
        its weights against oracle.paged's on the rows held here."""
        from minitorch_amd import device
        from oracle import paged as ref

        c, n = self.c, np.broadcast_to(n, self.c.batch)
        c.reserve(n)
        for i in range(c.n_layer):
            k, v = (self.rng.standard_normal((c.batch, c.n_head, n.max(), c.head_dim), dtype=np.float32)
                    for _ in range(2))
            q = (2 * self.rng.standard_normal((c.batch, H, 1, c.head_dim))).astype(np.float32)
            c.append(i, *(device.from_host(x, np.float32).t for x in (k, v)))
            was = None if c.weights is None else c.weights[i].numpy().astype(np.float64)
            got = c.attend(i, device.from_host(q, np.float32).t, 0.2).numpy()
            for b in range(c.batch):
                if not n[b]:
                    assert not got[b].any()
                    continue
                for rows, new in ((self.k, k), (self.v, v)):
                    rows[i][b] = np.concatenate([rows[i][b], new[b, :, :n[b]]], 1)
                L = self.k[i][b].shape[1]
                o, _, w, _, pv = ref.decode(q[b:b + 1], self.k[i][b][None], self.v[i][b][None],
                                            np.zeros((1, 1), np.int32), np.array([L]), 0.2)
                # a score is off by (D + 8) u of scale sum|q k|, some 12: 3e-5, and what
                # comes of it by twice that
                assert np.abs(got[b] - o[0]).max() <= 1e-4 * (1 + pv.max())
                if was is not None:
                    now = c.weights[i].numpy()[b]
                    assert np.abs(now[:, :L] - was[b, :, :L] - w[0]).max() <= 1e-4 * H
                    assert not now[:, L:].any()

    def cut(self, keep, recent):
        """The rows that a cut should keep, by the weights the cache holds."""
        self.w = [w.numpy() for w in self.c.weights]
        for i in range(self.c.n_layer):
            for b in range(self.c.batch):
                n = self.k[i][b].shape[1]
                kept = []
                for h in range(self.c.n_head):
                    at = np.arange(n)
                    if n > keep:
                        old = np.argsort(-self.w[i][b, h, :n - recent], kind="stable")[:keep - recent]
                        at = np.concatenate([np.sort(old), np.arange(n - recent, n)])
                    kept.append(at)
                    w = self.w[i][b, h, at]
                    self.w[i][b, h] = 0
                    self.w[i][b, h, :len(at)] = w
                for rows in (self.k, self.v):
                    rows[i][b] = np.stack([rows[i][b][h, at] for h, at in enumerate(kept)])

    def check(self):
        c = self.c
        assert [c.length(b) for b in range(c.batch)] == [x.shape[1] for x in self.k[0]]
        assert c.lengths.numpy().tolist() == [x.shape[1] for x in self.k[0]]
        assert np.array_equal(c.table.numpy(), c._tab)
        assert sorted(c._free + [int(i) for i in c._tab.ravel() if i >= 0]) == list(range(c.n_pages))
        for i in range(c.n_layer):
            assert np.array_equal(c.weights[i].numpy(), self.w[i])
            for pool, rows in ((c.k[i].numpy(), self.k[i]), (c.v[i].numpy(), self.v[i])):
                for b, x in enumerate(rows):
                    n = x.shape[1]
                    ids = c._tab[b, :-(-n // c.page)]
                    assert (ids >= 0).all()
                    held = pool[ids].transpose(1, 0, 2, 3).reshape(c.n_head, -1, c.head_dim)
                    assert np.array_equal(held[:, :n], x)


@pytest.mark.parametrize("pages,groups", [(None, 1), (20, 2), (17, 3)])
def test_trim_cuts_the_long_sequences_alone(dev, pages, groups):
    """Ragged lengths, three layers, three cuts after one another, in pools with
    room for all sequences at once, for two and for one: every layer's rows,
    weights and attention against the plain forms; sequences of `keep` rows or
    fewer stay in their pages."""
    import minitorch_amd as mt
    from minitorch_amd import kernels as K

    keep, recent, page, H = 12, 4, 4, 4
    c = mt.PagedKVCache(3, 2, 32, 4, 24, page=page, keep=keep, recent=recent, slack=3, pages=pages)
    s = Shadow(c, np.random.default_rng(41))
    s.step([14, 5, 12, 13], H)
    s.step(1, H)
    assert not c.trim()  # 15 rows at most
    for i in range(3):
        s.step([1, 0, 0, 1], H)
        if i:
            assert not c.trim()
            s.step([2, 0, 2, 2], H)
        long, pages_before = c._len > keep, c._tab.copy()
        calls, evict = [], K.kv_evict_paged
        try:
            K.kv_evict_paged = lambda *a, **kw: calls.append(1) or evict(*a, **kw)
            s.cut(keep, recent)
            assert c.trim() and not c.trim()
        finally:
            K.kv_evict_paged = evict
        assert long.any() and not long.all()
        if i == 0:
            assert len(calls) == 3 * groups
        s.check()
        assert np.array_equal(c._tab[~long], pages_before[~long])
        s.step(1, H)


def test_trim_in_a_pool_that_cannot_hold_all_cuts_at_once(dev):
    """Two sequences of 22 rows in 6 of 8 pages: their cuts take 2 pages each,
    and the first one's frees 3."""
    import minitorch_amd as mt

    c = mt.PagedKVCache(2, 2, 32, 2, 32, page=8, keep=16, recent=4, slack=5, pages=8)
    s = Shadow(c, np.random.default_rng(42))
    s.step(22, 2)
    s.cut(16, 4)
    assert c.trim()
    s.check()
    s.step(1, 2)
    # and where there is no room for a single one nothing has changed
    c = mt.PagedKVCache(1, 2, 32, 2, 32, page=8, keep=16, recent=4, slack=5, pages=7)
    c.reserve(22)
    before = state(c)
    with pytest.raises(RuntimeError, match="2 pages needed, 1 free"):
        c.trim()
    assert state(c) == before
    c.release(1)
    assert c.trim() and c.length(0) == 16


def test_generate_refuses_what_a_cache_cannot_hold_before_any_work(dev):
    m = model()
    idx = np.random.default_rng(43).integers(0, 50, (2, 10))

    def refused(error, match, n, **options):
        c = m.paged_cache(2, page=8, **options)
        before = state(c)
        with pytest.raises(error, match=match):
            m.generate(idx, n, cache=c)
        assert state(c) == before
        return c

    refused(ValueError, "exceed", 16, max_tokens=24)  # 25 rows at the end
    c = refused(RuntimeError, "pages", 24, pages=8)  # 33 rows, in 5 pages each
    np.random.seed(4)
    want = m.generate(idx, 23)
    np.random.seed(4)
    assert np.array_equal(m.generate(idx, 23, cache=c), want)  # 32, in 4
    # at most 17 rows a sequence in 3 pages each, and 2 for a cut
    options = dict(max_tokens=24, keep=12, slack=4)
    refused(RuntimeError, "pages", 30, pages=7, **options)
    np.random.seed(4)
    want = m.generate(idx, 30, cache=m.paged_cache(2, page=8, **options))
    np.random.seed(4)
    assert np.array_equal(m.generate(idx, 30, cache=m.paged_cache(2, page=8, pages=8, **options)), want)


def test_token_logprobs_temperatures(dev):
    """Hidden tokens have probability 0 up to the largest temperature; beyond
    it, where the others' 1 / temperature is no longer large beside that of
    -inf's stand-in, and where it overflows, the call is refused."""
    import minitorch_amd as mt

    x = np.array([[1.0, -np.inf, 2.0, -np.inf, 0.5]], np.float32)
    lp, ent, _, tops = mt.F.token_logprobs(mt.Tensor(x), [0], top=5, temperature=1e27)
    assert abs(float(lp.numpy()[0]) + np.log(3)) < 1e-6 and abs(float(ent.numpy()[0]) - np.log(3)) < 1e-6
    assert np.isneginf(tops.numpy()[0, 3:]).all()
    lp, ent, _, _ = mt.F.token_logprobs(mt.Tensor(x), [2], temperature=1e-38)
    assert float(lp.numpy()[0]) == 0 and float(ent.numpy()[0]) == 0
    for bad in (1e28, 1e30, 1e300, 0.9e-38, 5e-324):
        with pytest.raises(ValueError, match="temperature"):
            mt.F.token_logprobs(mt.Tensor(x), [0], temperature=bad)


def test_generate_with_bf16_pages_is_the_rounded_caches_model(dev):
    """The log probabilities of a generation through bf16 pages against the
    model's layers around an attention in 64 bits, whose steps see keys and values
    rounded to bf16 (a prompt's own positions see them in fp32)."""
    import minitorch_amd as mt
    from oracle.attention import bf16_round

    m = model()
    T0, n = 12, 20
    idx = np.random.default_rng(4).integers(0, 50, (2, T0))
    np.random.seed(6)
    ids, lp = m.generate(idx, n, cache=m.paged_cache(2, page=8, dtype="bfloat16"), return_logprobs=True)
    T, H, D = T0 + n - 1, 2, 32
    with mt.no_grad():
        x = m.tok_emb(ids[:, :T]) + m.pos_emb(np.arange(T))
        for block in m.blocks:
            h, a = block.ln1(x), block.attn
            q, k, v = (p(h).data.numpy().astype(np.float64).reshape(2, T, H, D).transpose(0, 2, 1, 3)
                       for p in (a.q_proj, a.k_proj, a.v_proj))
            o = np.zeros((2, H, T, D))
            for t in range(T):
                ks, vs = (y[:, :, :t + 1] if t < T0 else bf16_round(y[:, :, :t + 1].astype(np.float32)).astype(float)
                          for y in (k, v))
                s = np.matmul(ks, q[:, :, t, :, None])[..., 0] / np.sqrt(D)
                p = np.exp(s - s.max(-1, keepdims=True))
                o[:, :, t] = np.matmul((p / p.sum(-1, keepdims=True))[:, :, None], vs)[:, :, 0]
            x = x + a.out_proj(mt.Tensor(o.transpose(0, 2, 1, 3).reshape(2, T, H * D).astype(np.float32)))
            x = x + block.mlp(block.ln2(x))
        y = m.lm_head(m.ln_f(x)).data.numpy().astype(np.float64)[:, T0 - 1:]
    y = y - y.max(-1, keepdims=True)
    y = y - np.log(np.exp(y).sum(-1, keepdims=True))
    assert np.abs(lp - np.take_along_axis(y, ids[:, T0:, None], -1)[..., 0]).max() <= 1e-4


def test_rows_reserved_twice_and_never_written_are_all_taken_back(dev):
    """A refusal after two calls of reserve without a layer's append between
    leaves neither's rows; once layers have written, only the last ones'."""
    m = model()
    rng = np.random.default_rng(35)
    c = m.paged_cache(2, page=4)
    before = state(c)
    for n in (3, [2, 4]):
        c.reserve(n)
    with pytest.raises(ValueError, match="empty sequences"):
        run_paged(m, c, rng.integers(0, 50, (2, 4)), [0, 0])
    assert state(c) == before
    c.reserve(5)
    run_paged(m, c, rng.integers(0, 50, (2, 5)), [0, 0])
    before = state(c)
    for n in (1, 1, [0, 7]):
        c.reserve(n)
    c.undo()
    assert state(c) == before and c.length(0) == 5
    c.reserve(1)
    run_paged(m, c, rng.integers(0, 50, (2, 1)), [5, 5])
    c.undo()
    assert state(c) == before
