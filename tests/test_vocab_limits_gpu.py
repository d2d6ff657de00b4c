"""The operators of training with a large vocabulary at the ends of their ranges,
against the float64 forms (oracle.vocab)."""
import numpy as np
import pytest
from devarrays import T as dev_array, empty, full
from test_vocab_gpu import B, host, inside, rounded, tokens

from oracle import vocab as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,at", [((1 << 32) + 8, 0), ((1 << 31) + 1, 1)])
def test_dropout_of_one_row_longer_than_32_bits(dev, n, at):
    """The begin, the borders and the end of one row of n values are those of short
    calls that start there; `at` values into memory the row is taken value by value."""
    from minitorch_amd import kernels as K

    x = full((1, n + at), 1.0, "bfloat16")[:, at:]
    y = K.dropout(x, 0.5, 3, 11, out=x).view(n)
    for e in (0, (1 << 31) - 64, n // 2 // 4 * 4, n // 4 * 4 - 64):
        some = min(64, n - e)
        part = K.dropout(full((1, some), 1.0, "bfloat16"), 0.5, 3, 11 + e // 4)
        assert np.array_equal(host(y[e:e + some]), host(part)[0])
    # nothing is left as it was: every value is 0 or 2, the tail too
    assert set(np.unique(host(y[n - 8:]))) <= {0.0, 2.0}


def test_dropout_function_of_more_than_32_bits_of_values(dev):
    """F.dropout, which takes its tensor as one row, and its backward."""
    from minitorch_amd import F, Tensor
    from minitorch_amd import device as D
    from minitorch_amd import kernels as K

    n = (1 << 32) + 8
    x = Tensor(D.full((n,), 1.0), requires_grad=True)
    F.set_dropout_seed(9)
    y = F.dropout(x, 0.5)
    y.grad = D.full((n,), 3.0)
    y._backward()
    for e in (0, 1 << 31, n - 64):
        part = host(K.dropout(full((1, 64), 1.0), 0.5, 9, e // 4, subsequence=1))[0]
        assert np.array_equal(host(y.data.t[e:e + 64]), part)
        assert np.array_equal(host(x.grad.t[e:e + 64]), 3 * part)


# ---------------------------------------------------------------------------
# projection and cross-entropy: the bits of bf16 gradients
# ---------------------------------------------------------------------------

def _bf16_case(n, C, V, seed=0):
    rng = np.random.default_rng(seed + n + C + V)
    x = rounded(rng.standard_normal((n, C)), "bfloat16")
    w = rounded(rng.standard_normal((C, V)) * 2 / np.sqrt(C), "bfloat16")
    return x, w, tokens(rng, n, V)


def _bf16_bounds(x, w, r):
    """xent_bounds of bf16 outputs whose logits' gradient is off by 2^-18 of each entry
    in place of 2^-8: what fp32 gradients of the same call are off by, with 2^-18 of
    the entries, and the rounding of the result, 2^-8."""
    from test_vocab_gpu import xent_bounds

    dx, dw = xent_bounds(x, w, None, r, "bfloat16", "float32")[3:5]
    d = np.abs(r["dz"])
    dx, dw = dx + 2.0 ** -18 * (d @ np.abs(w).T), dw + 2.0 ** -18 * (np.abs(x).T @ d)
    return dx + B * (np.abs(r["dx"]) + dx), dw + B * (np.abs(r["dw"]) + dw)


# a wave a row, a workgroup a row, the longest rows; one block of rows and several; the
# small vocabularies' way
@pytest.mark.parametrize("n,C,V,more", [(60, 64, 40, {}), (130, 96, 700, {}), (300, 40, 5003, {}), (20, 24, 70001, {}),
                                        (300, 64, 136, dict(logits_bytes=100 * 136 * 4)), (600, 64, 65, {})])
def test_bf16_gradients_are_off_by_their_own_rounding(dev, n, C, V, more):
    from minitorch_amd import kernels as K

    x, w, labels = _bf16_case(n, C, V)
    r = ref.linear_xent(x, w, labels)
    bx, bw = _bf16_bounds(x, w, r)
    for tied in (False, True):
        args = dev_array(x, "bfloat16"), dev_array(w.T, "bfloat16").t() if tied else dev_array(w, "bfloat16")
        dx, dw = empty((n, C), "bfloat16"), empty((V, C) if tied else (C, V), "bfloat16")
        K.linear_xent(*args, dev_array(labels, "int64"), dx=dx, dw=dw.t() if tied else dw, **more)
        inside(host(dx), r["dx"], bx)
        inside(host(dw).T if tied else host(dw), r["dw"], bw)


def test_bf16_gradients_of_one_piece(dev):
    """On request from the logits' gradient in bf16: other values, inside the bounds that
    grant its rounding too."""
    from minitorch_amd import kernels as K
    from test_vocab_gpu import xent_bounds

    n, C, V = 130, 96, 700
    x, w, labels = _bf16_case(n, C, V)
    r = ref.linear_xent(x, w, labels)
    bounds = xent_bounds(x, w, None, r, "bfloat16", "bfloat16")[3:5]
    got = {}
    for one in (False, True):
        for more in ({}, dict(logits_bytes=64 * 704 * 4)):
            dx, dw = empty((n, C), "bfloat16"), empty((C, V), "bfloat16")
            K.linear_xent(dev_array(x, "bfloat16"), dev_array(w, "bfloat16"), dev_array(labels, "int64"), dx=dx, dw=dw,
                          one_piece=one, **more)
            inside(host(dx), r["dx"], bounds[0])
            inside(host(dw), r["dw"], bounds[1])
        got[one] = host(dx)
    assert not np.array_equal(got[False], got[True])


# ---------------------------------------------------------------------------
# projection and cross-entropy: logits as large as fp32 holds
# ---------------------------------------------------------------------------

# the small vocabularies' way, a wave a row, a workgroup a row, the longest rows
ROW_WAYS = [(300, 40, 65), (40, 24, 200), (20, 24, 3000), (20, 16, 10000), (9, 16, 30000), (9, 16, 50000), (9, 16, 70001)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kind", ["lowest", "highest", "both"])
@pytest.mark.parametrize("n,C,V", ROW_WAYS)
def test_linear_xent_of_logits_at_the_ends_of_fp32(dev, n, C, V, kind, dtype):
    """A mask of the type's lowest value that leaves nothing, logits near the highest,
    and both in one row.  Beside a bias of 3e38 the products vanish (its steps are 2e31):
    the k entries that hold the maximum have probability 1 / k, the others 0, exactly but
    for the rounding of 1 / k and of the steps to dz."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(n + V)
    x, w = rounded(rng.standard_normal((n, C)), dtype), rounded(rng.standard_normal((C, V)), dtype)
    low = float(np.finfo(np.float32).min)
    b = {"lowest": np.full(V, low), "highest": np.full(V, 3e38),
         "both": np.where(np.arange(V) % 3 == 1, low, 3e38)}[kind].astype(np.float32)
    labels = tokens(rng, n, V)
    some = (labels >= 0) & (labels < V)
    labels = np.where(some, labels // 3 * 3, labels)  # of the entries that are seen
    top = b.max()
    k = int((b == top).sum())
    dx, dw, db = empty((n, C)), empty((C, V)), empty((V,))
    args = [dev_array(x, dtype), dev_array(w, dtype), dev_array(labels, "int64")]
    U = 2.0 ** -24
    for grads in (dict(), dict(dx=dx, dw=dw, db=db)):
        loss, row, lse = K.linear_xent(*args, bias=dev_array(b), **grads)
        inside(host(lse), float(top) + np.log(k), 2 * U * abs(float(top)))
        # log k: the log's rounding and that of a sum of k ones, which is exact
        inside(host(row), np.where(some, np.log(k), 0.0), 4 * U * np.log(k))
        inside(host(loss), np.array([np.log(k)]), (n + 8) * U * np.log(k))
    count = some.sum()
    dz = np.where(b == top, 1.0 / k, 0.0) * np.ones((n, 1))
    dz[np.nonzero(some)[0], labels[some]] -= 1.0
    dz[~some] = 0.0
    dz /= count
    cut = 2.0 ** -22 if dtype == "float32" else 0.0
    size, xa, wa = np.abs(dz), np.abs(x.astype(np.float64)), np.abs(w.astype(np.float64))
    ed = 6 * U * (size + 1.0 / k / count)  # beside 1, 1 / k is off by a step of 1
    inside(host(dx), dz @ w.astype(np.float64).T, ed @ wa.T + ((V + 4) * U + cut) * (size @ wa.T))
    inside(host(dw), x.astype(np.float64).T @ dz, xa.T @ ed + ((n + 4) * U + cut) * (xa.T @ size))
    inside(host(db), dz.sum(0), ed.sum(0) + (n + 4) * U * size.sum(0))


# ---------------------------------------------------------------------------
# the table's gradient: small tables under many tokens
# ---------------------------------------------------------------------------

# chunks of one and of several groups of 64 tokens, the last one short; tables of as many
# values as take this way, and of more
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,V,C", [(140000, 65, 5), (140001, 10, 70), (200063, 128, 24), (70000, 255, 130), (66000, 65, 300),
                                   (40000, 192, 192), (40000, 193, 192)])
def test_lookup_grad_of_many_tokens(dev, n, V, C, dtype):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(n + V + C)
    ids = tokens(rng, n, V)
    g = rounded(rng.standard_normal((n, C)).astype(np.float32), dtype)
    counts = np.bincount(ids[(ids >= 0) & (ids < V)], minlength=V)[:, None]
    want, size = ref.lookup_grad(ids, g, V, 0.5)
    bound = (counts + 2) * 2.0 ** -24 * size
    dg, di = dev_array(g, dtype), dev_array(ids, "int64")
    first = host(K.embedding_grad(di, dg, full((V, C), 7.0), scale=0.5))
    inside(first, want, bound)
    assert np.array_equal(host(K.embedding_grad(di, dg, empty((V, C)), scale=0.5)), first)
    old = rng.standard_normal((V, C)).astype(np.float32)
    got = host(K.embedding_grad(di, dg, dev_array(old), scale=0.5, accumulate=True))
    inside(got, want + old, bound + 2.0 ** -24 * (np.abs(want + old) + bound))
    bad = int(np.nonzero((ids >= 0) & (ids < V))[0][-1])  # NaN stays in its token's row
    g[bad] = np.nan
    got = host(K.embedding_grad(di, dev_array(g, dtype), empty((V, C)), scale=0.5))
    rest = np.arange(V) != ids[bad]
    assert np.array_equal(got[rest], first[rest]) and np.isnan(got[ids[bad]]).all()


# ---------------------------------------------------------------------------
# projection and cross-entropy: either side of the small vocabularies' borders
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("n,C,V", [(1, 1024, 32), (5, 1025, 32), (40, 256, 33), (40, 257, 96), (300, 384, 80), (300, 385, 80),
                                   (70, 512, 64), (70, 513, 64), (3100, 513, 70), (50, 384, 81), (4200, 1030, 20)])
def test_linear_xent_where_the_small_vocabularies_way_ends(dev, n, C, V, dtype, out):
    from test_vocab_gpu import check_xent

    check_xent(n, C, V, dtype, out, tied=n % 2 == 0)


# ---------------------------------------------------------------------------
# dropout: probability 0
# ---------------------------------------------------------------------------

# Philox's output words below 256, whose uniform is 0: (seed, counter, word)
ZEROS = [(5, 2920362, 1), (6, 2977858, 3)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("seed,counter,word", ZEROS)
def test_dropout_of_probability_0_is_the_identity(dev, seed, counter, word, dtype):
    """Where the uniform is 0 too: in whole vectors, value by value, with a residual."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(seed)
    x, r = (rounded(rng.standard_normal((2, 64)), dtype) for _ in range(2))
    # (the oracle's mask lacks that value: the case is the one it is meant to be)
    assert (~ref.keep((2, 64), 0.0, seed, counter - 3)).nonzero()[1].tolist() == [12 + word]
    for cols in (64, 63):
        dx = dev_array(x, dtype)[:, :cols]
        got = K.dropout(dx, 0.0, seed, counter - 3, out=empty((2, 64), dtype)[:, :cols])
        assert np.array_equal(host(got), x[:, :cols])
        got = K.dropout(dx, 0.0, seed, counter - 3, residual=dev_array(r, dtype)[:, :cols], out=empty((2, 64), dtype)[:, :cols])
        assert np.array_equal(host(got), rounded(r + x, dtype)[:, :cols])
    # and the smallest probabilities drop it, and no other
    got = host(K.dropout(full((2, 64), 1.0, dtype), 2.0 ** -30, seed, counter - 3))
    assert np.argwhere(got == 0).tolist() == [[0, 12 + word]]


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("n,C,V,rows", [(5, 40, 65, 1), (22, 40, 65, 7), (530, 70, 20, 256), (262144 + 77, 8, 20, 1 << 30)])
def test_linear_xent_small_vocabularies_in_blocks_of_few_rows(dev, n, C, V, rows, dtype, out):
    """Blocks of one row, of a few, of as many as there may be (2^18)."""
    from test_vocab_gpu import check_xent

    check_xent(n, C, V, dtype, out, tied=n % 2 == 1, logits_bytes=rows * (-(-V // 32) * 32) * 4)
