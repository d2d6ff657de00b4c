"""Training with a large vocabulary on the GPU against the plain float64 forms
(oracle.vocab): the scaled lookup and its gradient, dropout without a mask, the
projection with its cross-entropy and gradients.

Bounds, with u = 2^-24 and b = 2^-8 (half a step of bf16): a product is off by u,
a sum of k terms by (k + 1) u of the terms' magnitudes, a value stored in bf16 by b
of its own."""
import numpy as np
import pytest
from devarrays import T as dev_array, empty, full

from oracle import vocab as ref
from oracle.attention import bf16_round

pytestmark = pytest.mark.gpu
U, B = 2.0 ** -24, 2.0 ** -8


def host(t):
    """A device array's values; those of rows that lie apart too (in memory that
    `wide` or a whole sheet holds)."""
    t = getattr(t, "t", t) if not callable(getattr(t, "t", None)) else t
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) > t.shape[1] and t.shape[0]:
        return t.as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1)).numpy()[:, :t.shape[1]]
    return t.numpy()


def rounded(x, dtype):
    x = np.asarray(x, np.float32)
    return bf16_round(x) if dtype == "bfloat16" else x


def tokens(rng, n, V, none=0.2):
    """Ids whose frequencies fall as words' do, some of them outside [0, V)."""
    ids = rng.permutation(V)[np.minimum(np.exp(rng.random(n) * np.log(V + 1)).astype(int) - 1, V - 1)]
    bad = rng.random(n) < none
    ids[bad] = rng.choice([-1, -(1 << 40), V, V + 7, 1 << 40], bad.sum())
    return ids.astype(np.int64)


def wide(x, dtype, pad, at=0):
    """x as a view whose rows lie `pad` values apart, `at` values into its memory."""
    rows, cols = x.shape
    mem = np.full(rows * (cols + pad) + at, np.nan, np.float32)
    mem[at:].reshape(rows, cols + pad)[:, :cols] = x
    return dev_array(mem, dtype)[at:].view(rows, cols + pad)[:, :cols]


def inside(got, want, bound):
    with np.errstate(invalid="ignore"):
        ok = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= bound)
    assert ok.all(), (int((~ok).sum()), float(np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300))))


# ---------------------------------------------------------------------------
# lookup
# ---------------------------------------------------------------------------
LOOKUPS = [
    (1, 1, 1, 0, 0), (3, 2, 5, 0, 0), (64, 65, 384, 0, 0), (500, 1000, 64, 3, 1), (257, 300, 1023, 1, 0),
    (40, 11, 8192, 0, 0), (1000, 5003, 96, 8, 8), (7, 9, 4, 0, 3), (130, 70, 20, 4, 4),
]


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,V,C,pad,at", LOOKUPS)
def test_lookup(dev, n, V, C, pad, at, dtype, out):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(n * 31 + C)
    w, ids = rounded(rng.standard_normal((V, C)), dtype), tokens(rng, n, V)
    for scale in (1.0, 19.596):
        mem = full((n, C + pad), 7.0, "float32") if out == "float32" else dev_array(np.full((n, C + pad), 7.0), out)
        got = host(K.embedding_lookup(wide(w, dtype, pad, at), dev_array(ids, "int64"), scale=scale, out=mem[:, :C]))
        want = ref.lookup(w, ids, float(np.float32(scale)))
        inside(got, want, (U if out == "float32" else U + B * (1 + U)) * np.abs(want))
        assert (host(mem)[:, C:] == 7.0).all()
        assert (got[(ids < 0) | (ids >= V)] == 0).all()


def test_lookup_of_nothing(dev):
    from minitorch_amd import kernels as K

    assert host(K.embedding_lookup(dev_array(np.ones((3, 4))), empty((0,), "int64"))).shape == (0, 4)


def test_lookup_keeps_what_is_not_finite(dev):
    from minitorch_amd import kernels as K

    w = np.array([[np.inf, -np.inf, np.nan, 3e38], [np.nan] * 4], np.float32)
    got = host(K.embedding_lookup(dev_array(w), dev_array(np.array([0, -1]), "int64"), scale=2.0))
    assert np.array_equal(got, [[np.inf, -np.inf, np.nan, np.inf], [0, 0, 0, 0]], equal_nan=True)


# ---------------------------------------------------------------------------
# its gradient
# ---------------------------------------------------------------------------
GRADS = [
    (1, 1, 1), (2, 7, 3), (63, 65, 384), (64, 1, 64), (65, 2, 130), (300, 5003, 96), (1025, 3, 257),
    (4096, 256, 32), (4097, 257, 33), (9000, 65537, 8), (20000, 65, 16), (12345, 70000, 5), (8191, 40, 1000),
]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,V,C", GRADS)
def test_lookup_grad(dev, n, V, C, dtype):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(n + V + C)
    g, ids = rounded(rng.standard_normal((n, C)), dtype), tokens(rng, n, V)
    counts = np.bincount(ids[(ids >= 0) & (ids < V)], minlength=V)[:, None]
    old = rng.standard_normal((V, C + 3)).astype(np.float32)
    for scale, pad, acc in ((1.0, 0, False), (19.596, 5, True)):
        mem = dev_array(old)
        K.embedding_grad(dev_array(ids, "int64"), wide(g, dtype, pad, pad), mem[:, :C], scale=scale, accumulate=acc)
        want, size = ref.lookup_grad(ids, g, V, float(np.float32(scale)))
        bound = (counts + 2) * U * size
        got = host(mem)
        if acc:
            assert np.array_equal(got[:, :C][counts[:, 0] == 0], old[:, :C][counts[:, 0] == 0])
            want = want + old[:, :C]
            bound = bound + U * (np.abs(want) + bound)
        inside(got[:, :C], want, bound)
        assert np.array_equal(got[:, C:], old[:, C:])


@pytest.mark.parametrize("V,which", [(5, 3), (70000, 69999), (70000, 0)])
def test_lookup_grad_of_one_token(dev, V, which):
    """All rows belong to one token, or to none."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(V + which)
    n, C = 9001, 12
    g = rng.standard_normal((n, C)).astype(np.float32)
    for ids in (np.full(n, which), np.full(n, -1)):
        dw = full((V, C), 7.0)
        K.embedding_grad(dev_array(ids, "int64"), dev_array(g), dw)
        want, size = ref.lookup_grad(ids, g, V)
        inside(host(dw), want, (n + 2) * U * size)


def test_lookup_grad_of_no_tokens(dev):
    from minitorch_amd import kernels as K

    for acc, want in ((False, 0.0), (True, 7.0)):
        dw = full((300, 6), 7.0)
        K.embedding_grad(empty((0,), "int64"), empty((0, 6)), dw, accumulate=acc)
        assert (host(dw) == want).all()


def test_lookup_grad_rows_without_a_token_may_hold_anything(dev):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(3)
    ids = tokens(rng, 700, 50, 0.5)
    g = rng.standard_normal((700, 40)).astype(np.float32)
    bad = g.copy()
    bad[(ids < 0) | (ids >= 50)] = np.nan
    a, b = (K.embedding_grad(dev_array(ids, "int64"), dev_array(x), empty((50, 40))) for x in (g, bad))
    assert np.array_equal(host(a), host(b))


@pytest.mark.parametrize("n,V,C", [(20000, 65, 16), (9000, 65537, 8)])
def test_lookup_grad_same_bits_every_time(dev, n, V, C):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(5)
    ids, g = dev_array(tokens(rng, n, V), "int64"), dev_array(rng.standard_normal((n, C)))
    first = host(K.embedding_grad(ids, g, empty((V, C))))
    for _ in range(5):
        assert np.array_equal(host(K.embedding_grad(ids, g, empty((V, C)))), first)


# tokens, table rows, width: few tokens of wide and narrow rows and the borders where that
# ends, small tables up to their largest and to their shortest batch, and what lies behind
GRAD_WAYS = [(4096, 3, 64), (4097, 3, 64), (2048, 40, 128), (2048, 40, 129), (100, 9, 2621), (100, 9, 2622), (4096, 50000, 1),
             (4096, 127, 70), (8192, 255, 40), (8191, 255, 40), (12001, 200, 515), (8200, 256, 24), (5000, 128, 1030),
             (1024, 9, 300), (1025, 9, 300), (1000, 700, 1300), (1024, 1, 520)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,V,C", GRAD_WAYS)
def test_lookup_grad_borders(dev, n, V, C, dtype):
    """Added up and written; NaN and infinities reach the row of their own token alone;
    no token at all."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(n + V + C)
    g, ids = rounded(rng.standard_normal((n, C)), dtype), tokens(rng, n, V)
    counts = np.bincount(ids[(ids >= 0) & (ids < V)], minlength=V)[:, None]
    want, size = ref.lookup_grad(ids, g, V, 0.5)
    bound = (counts + 2) * U * size
    dg, di = dev_array(g, dtype), dev_array(ids, "int64")
    inside(host(K.embedding_grad(di, dg, full((V, C), 7.0), scale=0.5)), want, bound)
    old = rng.standard_normal((V, C)).astype(np.float32)
    got = host(K.embedding_grad(di, dg, dev_array(old), scale=0.5, accumulate=True))
    inside(got, want + old, bound + U * (np.abs(want + old) + bound))
    assert np.array_equal(got[counts[:, 0] == 0], old[counts[:, 0] == 0])
    plain = host(K.embedding_grad(di, dg, empty((V, C))))
    at = np.nonzero((ids >= 0) & (ids < V))[0][:2]
    bad = g.copy()
    bad[at[0]], bad[at[1], 0] = np.nan, np.inf
    got = host(K.embedding_grad(di, dev_array(bad, dtype), empty((V, C))))
    rest = np.setdiff1d(np.arange(V), ids[at])
    assert np.array_equal(got[rest], plain[rest])
    assert np.isnan(got[ids[at[0]]]).all() and not np.isfinite(got[ids[at[1]], 0])
    none = dev_array(np.full(n, -1), "int64")
    assert not host(K.embedding_grad(none, dg, full((V, C), 7.0))).any()
    assert np.array_equal(host(K.embedding_grad(none, dg, dev_array(old), accumulate=True)), old)


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
DROPS = [(1, 1), (1, 3), (1, 5), (32, 64), (7, 129), (300, 384), (1000, 7), (33, 1030), (5, 8), (256, 2048)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", DROPS)
def test_dropout(dev, rows, cols, residual, dtype):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(rows + cols)
    x, r = (rounded(rng.standard_normal((rows, cols)), dtype) for _ in range(2))
    for p, seed, offset, sub, pad, at in ((0.1, 7, 0, 0, 0, 0), (0.5, (1 << 63) + 11, (1 << 32) - 2, 0, 0, 1),
                                          (0.9, 123456789123, (1 << 62) + 5, 3, 8, 0), (0.25, 5, 9, 1, 3, 3)):
        res = wide(r, dtype, pad, at) if residual else None
        out = wide(np.zeros_like(x), dtype, pad, at)
        K.dropout(wide(x, dtype, pad, at), p, seed, offset, residual=res, out=out, subsequence=sub)
        got = host(out)
        mask = ref.keep(x.shape, p, seed, offset, sub)
        scaled = np.where(mask, x * np.float32(1.0 / (1.0 - p)), np.float32(0))  # float32, as the kernel rounds
        want = rounded(r + scaled if residual else scaled, dtype)
        assert np.array_equal(got, want)


def test_dropout_has_the_keep_masks_of_the_fused_attention(dev):
    from minitorch_amd import kernels as K

    mask, _ = K.dropout_keep_philox((2, 3, 5, 8), 0.3, 99, 1234)
    got = host(K.dropout(full((30, 8), 1.0), 0.3, 99, 1234))
    assert np.array_equal(got != 0, host(mask).reshape(30, 8) != 0)


def test_dropout_in_place_and_added(dev):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(11)
    x, r = (rng.standard_normal((50, 77)).astype(np.float32) for _ in range(2))
    want = host(K.dropout(dev_array(x), 0.4, 1, 2))
    a = dev_array(x)
    K.dropout(a, 0.4, 1, 2, out=a)
    assert np.array_equal(host(a), want)
    b = dev_array(r)
    K.dropout(dev_array(x), 0.4, 1, 2, residual=b, out=b)
    assert np.array_equal(host(b), r + want)


def test_dropout_drops_what_is_not_finite(dev):
    from minitorch_amd import kernels as K

    mask = ref.keep((40, 40), 0.5, 3, 0)
    x = np.where(mask, 1.0, np.nan).astype(np.float32)
    got = host(K.dropout(dev_array(x), 0.5, 3, 0))
    assert np.array_equal(got, np.where(mask, 2.0, 0.0))


def test_dropout_base_is_read_when_it_runs(dev):
    from minitorch_amd import kernels as K

    x = full((9, 64), 1.0)
    base = dev_array(np.array([0]), "int64")
    for at in (0, 5, (1 << 33) + 1):
        base.copy_(np.array([at]))
        got = host(K.dropout(x, 0.5, 8, 100, base=base))
        assert np.array_equal(got != 0, ref.keep((9, 64), 0.5, 8, 100 + at))


@pytest.mark.parametrize("p", [0.0, float(np.float32(1) - np.float32(2) ** -24)])
def test_dropout_at_the_ends(dev, p):
    """p = 0 drops only the uniform 0, p just below 1 everything."""
    from minitorch_amd import kernels as K

    got = host(K.dropout(full((300, 300), 1.0), p, 21, 0)) != 0
    assert np.array_equal(got, ref.keep((300, 300), p, 21))
    assert got.all() if p == 0 else not got.any()


# ---------------------------------------------------------------------------
# projection and cross-entropy
# ---------------------------------------------------------------------------

def xent_bounds(x, w, bias, r, dtype, out):
    """Bounds of lse, row_loss, loss, dx, dw, db."""
    x, w = np.abs(np.asarray(x, np.float64)), np.abs(np.asarray(w, np.float64))
    n, C = x.shape
    V = w.shape[1]
    # fp32 products drop 2^-22 of the terms (three bf16 pieces), bf16 ones nothing
    cut = 2.0 ** -22 if dtype == "float32" else 0.0
    ez = ((C + 2) * U + cut) * (x @ w) + U * (np.abs(r["z"]) + (0 if bias is None else np.abs(bias)))
    seen = r["z"] > -1e30  # hidden entries have probability 0 whatever their error
    z = np.where(seen, np.abs(r["z"]), 0.0)
    ez = np.where(seen, ez, 0.0).max(1)
    mag = z.max(1)
    e = ez + U * (4 * mag + V + 16)  # a term exp(z - max) and the sum of V of them
    fin = np.where(np.isfinite(r["lse"]), np.abs(r["lse"]), 0.0)
    lse = e + 4 * U * (fin + mag)
    row = lse + ez + 4 * U * (fin + mag)
    # All entries of a row with a label, not those alone whose gradient is not 0: the
    # label's own is p - 1, exactly 0 in float64 once 1 - p < 2^-54 (or V is 1), and a p
    # that is off by p (2 e + 8 u) is off by that beside 1 too.
    named = r["some"]
    count = max(1, int(named.sum()))
    loss = row.sum() / count + (n + 4) * U * np.where(np.isfinite(r["row_loss"]), r["row_loss"], 0).sum() / count
    d = np.abs(r["dz"])
    ed = r["p"] * (2 * e + 8 * U)[:, None] * named[:, None] / count + 4 * U * d
    ed = ed + (B if out == "bfloat16" else U) * d if dtype == "bfloat16" else ed
    size = B if out == "bfloat16" else U
    dx = ed @ w.T + ((V + 2) * U + cut) * (d @ w.T)
    dw = x.T @ ed + ((n + 2) * U + cut) * (x.T @ d)
    db = (r["p"] * (2 * e + 8 * U)[:, None] / count + 4 * U * d).sum(0) + (n + 2) * U * d.sum(0)
    return lse, row, loss, dx + size * (np.abs(r["dx"]) + dx), dw + size * (np.abs(r["dw"]) + dw), db


def check_xent(n, C, V, dtype, out="float32", tied=False, bias=True, none=0.2, pad=0, at=0, seed=0, std=2.0, **more):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(seed + n + C + V)
    x = rounded(rng.standard_normal((n, C)), dtype)
    w = rounded(rng.standard_normal((C, V)) * std / np.sqrt(C), dtype)
    b = (0.5 * rng.standard_normal(V)).astype(np.float32) if bias else None
    labels = tokens(rng, n, V, none)
    r = ref.linear_xent(x, w, labels, b)
    lay = lambda m: wide(m.T, dtype, pad, at).t() if tied else wide(m, dtype, pad, at)  # noqa: E731
    args = (wide(x, dtype, pad, at), lay(w), dev_array(labels, "int64"))
    db = dev_array(b) if bias else None
    bounds = xent_bounds(x, w, b, r, dtype, out)
    def forward(outs):
        for g, want, bd in zip(outs, ([r["loss"]], r["row_loss"], r["lse"]), (bounds[2], bounds[1], bounds[0])):
            inside(host(g), np.asarray(want), bd)

    forward(K.linear_xent(*args, bias=db, **more))
    sheet = lambda s: dev_array(np.full((s[0], s[1] + pad), 7.0), out)  # noqa: E731
    mx, mw, mb = sheet((n, C)), sheet((V, C) if tied else (C, V)), full((V,), 7.0)
    dw = mw[:, :C].t() if tied else mw[:, :V]
    got = K.linear_xent(*args, bias=db, dx=mx[:, :C], dw=dw, db=mb if bias else None, **more)
    forward(got)
    inside(host(mx)[:, :C], r["dx"], bounds[3])
    hw = host(mw)
    inside(hw[:, :C].T if tied else hw[:, :V], r["dw"], bounds[4])
    assert (host(mx)[:, C:] == 7.0).all() and (hw[:, C if tied else V:] == 7.0).all()
    if bias:
        inside(host(mb), r["db"], bounds[5])
    return args, db, r


XENTS = [
    (1, 1, 1), (1, 8, 2), (3, 64, 65), (5, 7, 9), (64, 96, 130), (65, 33, 257), (130, 384, 65), (200, 130, 1000),
    (257, 64, 5003), (512, 256, 512), (300, 129, 1031), (70, 520, 2049), (1, 64, 70001), (9, 40, 66000),
]


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,C,V", XENTS)
def test_linear_xent(dev, n, C, V, tied, dtype, out):
    check_xent(n, C, V, dtype, out, tied=tied, bias=n % 2 == 1)


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("V", [256, 512, 513, 1024, 1025, 4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769, 40960,
                               40961, 65536, 65537])
def test_linear_xent_lengths_of_rows(dev, V, bias, dtype, out):
    """Where one way to walk a row ends and the next begins."""
    check_xent(5, 6, V, dtype, out, tied=True, bias=bias)


# many rows and a small vocabulary: one to six chunks of C, the borders of the tiles of
# 16 entries, rows that fill no group of 16 or 64, and what lies beside
NARROW = [(4, 1, 1), (20, 5, 3), (19, 5, 3), (63, 8, 16), (130, 32, 17), (300, 64, 32), (300, 65, 33), (515, 128, 64),
          (1030, 129, 65), (1025, 200, 65), (2000, 384, 65), (700, 130, 80), (129, 32, 81), (640, 33, 96), (515, 100, 96),
          (640, 130, 95), (640, 130, 97), (4100, 70, 65)]


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,C,V", NARROW)
def test_linear_xent_small_vocabularies(dev, n, C, V, tied, dtype, out):
    check_xent(n, C, V, dtype, out, tied=tied, bias=n % 2 == 0)


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
def test_linear_xent_small_vocabulary_strides_and_blocks(dev, dtype, out):
    for tied in (False, True):
        for pad, at in ((8, 0), (4, 4), (3, 1)):
            check_xent(210, 44, 65, dtype, out, tied=tied, pad=pad, at=at)
            check_xent(210, 37, 20, dtype, out, tied=tied, pad=pad, at=at)
        check_xent(1000, 40, 65, dtype, out, tied=tied, logits_bytes=256 * 96 * 4)
        check_xent(700, 20, 30, dtype, out, tied=tied, logits_bytes=100 * 32 * 4)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_xent_small_vocabulary_rows_far_apart(dev, dtype):
    """Rows of the weights 2^22 values apart."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(3)
    n, C, V, ld = 30, 3, 7, 1 << 22
    x, w = rounded(rng.standard_normal((n, C)), dtype), rounded(rng.standard_normal((C, V)), dtype)
    labels = tokens(rng, n, V)
    r = ref.linear_xent(x, w, labels)
    bd = xent_bounds(x, w, None, r, dtype, "float32")
    dx, dw = empty((n, C)), empty((C, V))
    loss, row, lse = K.linear_xent(dev_array(x, dtype), wide(w, dtype, ld - V), dev_array(labels, "int64"), dx=dx,
                                   dw=dw)
    for got, want, b in ((lse, r["lse"], bd[0]), (row, r["row_loss"], bd[1]), (dx, r["dx"], bd[3]), (dw, r["dw"], bd[4])):
        inside(host(got), want, b)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_xent_small_vocabulary_hidden_entries_and_rows(dev, dtype):
    """Entries hidden by a bias of -inf, all of a row's, rows without a label that hold
    anything finite; gradients wanted one at a time; the same bits every time."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(8)
    n, C, V = 300, 40, 65
    x, w = rounded(rng.standard_normal((n, C)), dtype), rounded(rng.standard_normal((C, V)) / 6, dtype)
    b = np.where(rng.random(V) < 0.4, -np.inf, 0.0).astype(np.float32)
    b[0] = 0.0
    labels = np.where(rng.random(n) < 0.3, -1, 0)
    x[labels < 0] = rounded(1e38, dtype)
    seen = x.copy()
    seen[labels < 0] = 0.0
    r = ref.linear_xent(seen, w, labels, b)
    bd = xent_bounds(seen, w, np.where(b == -np.inf, 0.0, b), r, dtype, "float32")
    args = [dev_array(x, dtype), dev_array(w, dtype), dev_array(labels, "int64")]
    first = None
    for _ in range(3):
        dx, dw, db = empty((n, C)), empty((C, V)), empty((V,))
        loss, row, lse = K.linear_xent(*args, bias=dev_array(b), dx=dx, dw=dw, db=db)
        now = [host(t) for t in (loss, row, dx, dw, db)]
        first = first or now
        assert all(np.array_equal(p, q) for p, q in zip(first, now))
    inside(host(lse)[labels >= 0], r["lse"][labels >= 0], bd[0][labels >= 0])
    for got, want, bound in zip(now, ([r["loss"]], r["row_loss"], r["dx"], r["dw"], r["db"]), (bd[2], bd[1], *bd[3:])):
        inside(got, np.asarray(want), bound)
    assert (now[4][b == -np.inf] == 0).all()
    for name, like, want in (("dx", (n, C), now[2]), ("dw", (C, V), now[3]), ("db", (V,), now[4])):
        g = empty(like)
        K.linear_xent(*args, bias=dev_array(b), **{name: g})
        assert np.array_equal(host(g), want)
    none = dev_array(np.full(V, -np.inf))
    dx, dw, db = empty((n, C)), empty((C, V)), empty((V,))
    args[0] = dev_array(seen, dtype)
    loss, row, lse = K.linear_xent(*args, bias=none, dx=dx, dw=dw, db=db)
    assert (host(lse) == -np.inf).all() and np.array_equal(host(row), np.where(labels < 0, 0, np.inf))
    assert abs(host(db)[0] + 1) <= (n + 2) * U and not host(db)[1:].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,C,V", [(1, 70, 5003), (2, 64, 4113), (17, 130, 9000), (64, 33, 20001), (65, 33, 20001), (65, 128, 65537),
                                   (72, 1031, 8201), (127, 420, 20003), (128, 130, 4999)])
def test_linear_xent_few_rows(dev, n, C, V, dtype):
    for tied in (False, True):
        check_xent(n, C, V, dtype, tied=tied)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("pad,at", [(8, 0), (3, 1), (1, 5)])
def test_linear_xent_strides(dev, pad, at, dtype):
    for tied in (False, True):
        check_xent(70, 48, 136, dtype, dtype, tied=tied, pad=pad, at=at)
        check_xent(33, 37, 301, dtype, "float32", tied=tied, pad=pad, at=at)


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("rows", [1, 7, 100, 256, 600])
def test_linear_xent_in_blocks_of_rows(dev, rows, tied, dtype, out):
    """Logits of a few rows at a time; the last block may be a single one."""
    n = {1: 5, 7: 22, 100: 201, 256: 513, 600: 700}[rows]
    check_xent(n, 40, 136, dtype, out, tied=tied, logits_bytes=rows * 136 * 4)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_xent_without_labels(dev, dtype):
    """No row has a label, or there are no rows: the loss and gradients are 0."""
    from minitorch_amd import kernels as K

    check_xent(40, 64, 100, dtype, none=1.0)
    x, w = empty((0, 6), dtype), dev_array(np.ones((6, 10)), dtype)
    dx, dw, db = empty((0, 6)), full((6, 10), 7.0), full((10,), 7.0)
    loss, row, lse = K.linear_xent(x, w, empty((0,), "int64"), bias=full((10,), 1.0), dx=dx, dw=dw, db=db)
    assert host(loss)[0] == 0 and host(row).shape == (0,) and not host(dw).any() and not host(db).any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_xent_hidden_entries(dev, dtype):
    """A bias of -inf, or of the type's lowest value, hides entries of the
    vocabulary; one that hides all of them but the label, or the label itself."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(9)
    n, C, V = 20, 32, 70
    x, w = rounded(rng.standard_normal((n, C)), dtype), rounded(rng.standard_normal((C, V)) / 4, dtype)
    for low in (-np.inf, float(np.finfo(np.float32).min)):
        b = np.where(rng.random(V) < 0.5, low, 0.0).astype(np.float32)
        b[:2] = 0.0, low
        for labels in (np.zeros(n, np.int64), np.where(np.arange(n) == 3, 1, 0)):
            r = ref.linear_xent(x, w, labels, b)
            dx, dw, db = empty((n, C)), empty((C, V)), empty((V,))
            loss, row, lse = K.linear_xent(dev_array(x, dtype), dev_array(w, dtype), dev_array(labels, "int64"),
                                           bias=dev_array(b), dx=dx, dw=dw, db=db)
            bd = xent_bounds(x, w, np.where(b == low, 0.0, b), r, dtype, "float32")
            inside(host(lse), r["lse"], bd[0])
            if low == -np.inf:
                inside(host(row), r["row_loss"], bd[1])
            else:
                inside(host(row), r["row_loss"], bd[1] + 4 * U * np.abs(r["row_loss"]))
            inside(host(dx), r["dx"], bd[3] + 1e-7)
            inside(host(dw), r["dw"], bd[4] + 1e-7)
            assert (host(db)[(b == low) & (np.arange(V) != 1)] == 0).all()


def test_linear_xent_all_hidden(dev):
    """Every logit -inf: lse -inf, row loss +inf, the label's own gradient alone."""
    from minitorch_amd import kernels as K

    x, w = np.ones((2, 4), np.float32), np.ones((4, 6), np.float32)
    dx, dw, db = empty((2, 4)), empty((4, 6)), empty((6,))
    loss, row, lse = K.linear_xent(dev_array(x), dev_array(w), dev_array(np.array([2, -1]), "int64"),
                                   bias=full((6,), -np.inf), dx=dx, dw=dw, db=db)
    assert (host(lse) == -np.inf).all() and np.array_equal(host(row), [np.inf, 0.0])
    assert np.array_equal(host(db), [0, 0, -1, 0, 0, 0]) and np.array_equal(host(dx), [[-1] * 4, [0] * 4])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_xent_rows_without_a_label_may_hold_anything(dev, dtype):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(4)
    n, C, V = 60, 40, 90
    x, w = rounded(rng.standard_normal((n, C)), dtype), rounded(rng.standard_normal((C, V)), dtype)
    labels = tokens(rng, n, V, 0.4)
    outs = []
    for row in (0.0, 1e38):  # finite, but their logits are not
        y = x.copy()
        y[(labels < 0) | (labels >= V)] = rounded(row, dtype)
        dx, dw = empty((n, C)), empty((C, V))
        loss, r, _ = K.linear_xent(dev_array(y, dtype), dev_array(w, dtype), dev_array(labels, "int64"), dx=dx, dw=dw)
        outs.append([host(t) for t in (loss, r, dx, dw)])
    for a, b in zip(*outs):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_xent_gradient_against_differences(dev, dtype):
    """The gradients against central differences of the float64 loss."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(2)
    n, C, V = 12, 20, 50
    x, w = rounded(rng.standard_normal((n, C)), dtype), rounded(rng.standard_normal((C, V)) / 3, dtype)
    b = rng.standard_normal(V).astype(np.float32)
    labels = tokens(rng, n, V)
    dx, dw, db = empty((n, C)), empty((C, V)), empty((V,))
    K.linear_xent(dev_array(x, dtype), dev_array(w, dtype), dev_array(labels, "int64"), bias=dev_array(b), dx=dx, dw=dw,
                  db=db)
    r = ref.linear_xent(x, w, labels, b)
    bd = xent_bounds(x, w, b, r, dtype, "float32")
    h = 1e-4
    for got, arg, bound in ((dx, 0, bd[3]), (dw, 1, bd[4]), (db, 2, bd[5])):
        d = rng.standard_normal(host(got).shape)
        vals = []
        for s in (h, -h):
            a = [x.astype(np.float64), w.astype(np.float64), b.astype(np.float64)]
            a[arg] = a[arg] + s * d
            vals.append(ref.linear_xent(a[0], a[1], labels, a[2])["loss"])
        slope = (vals[0] - vals[1]) / (2 * h)
        # h^2 times a third derivative of order (|d| |x|)^3, and 1e-16 / h of rounding
        assert abs(slope - float((host(got) * d).sum())) <= float((bound * np.abs(d)).sum()) + 1e-5


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
def test_linear_xent_same_bits_every_time(dev, dtype, out):
    from minitorch_amd import kernels as K

    args, db, _ = check_xent(300, 64, 2000, dtype, out)
    first = None
    for _ in range(4):
        dx, dw, d = empty((300, 64), out), empty((64, 2000), out), empty((2000,))
        r = K.linear_xent(*args, bias=db, dx=dx, dw=dw, db=d)
        now = [host(t) for t in (*r, dx, dw, d)]
        first = first or now
        assert all(np.array_equal(a, b) for a, b in zip(first, now))


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
def test_linear_xent_wanted_gradients_alone(dev, dtype, out):
    from minitorch_amd import kernels as K

    args, db, r = check_xent(50, 40, 210, dtype, out)
    full_ = [empty((50, 40), out), empty((40, 210), out), empty((210,))]
    K.linear_xent(*args, bias=db, dx=full_[0], dw=full_[1], db=full_[2])
    for i, name in enumerate(("dx", "dw")):
        g = empty(full_[i].shape, out)
        K.linear_xent(*args, bias=db, **{name: g})
        assert np.array_equal(host(g), host(full_[i]))
    # db alone may be added up in another order: two sums of the 50 rows' terms, each off
    # by at most 52 roundings of their magnitudes
    d = empty((210,))
    K.linear_xent(*args, bias=db, db=d)
    inside(host(d), host(full_[2]), 2 * 52 * U * np.abs(r["dz"]).sum(0))


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("n,C,V", [(70, 40, 300), (500, 40, 65)])
def test_linear_xent_gradient_in_the_other_order(dev, n, C, V, dtype, out):
    """The weights' gradient laid out as the transpose of the weights."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(n)
    x, w = rounded(rng.standard_normal((n, C)), dtype), rounded(rng.standard_normal((C, V)) / 6, dtype)
    labels = tokens(rng, n, V)
    r = ref.linear_xent(x, w, labels)
    bound = xent_bounds(x, w, None, r, dtype, out)[4]
    for tied in (False, True):
        wd = dev_array(w.T, dtype).t() if tied else dev_array(w, dtype)
        dw = empty((C, V), out) if tied else empty((V, C), out).t()
        K.linear_xent(dev_array(x, dtype), wd, dev_array(labels, "int64"), dw=dw)
        inside(host(dw) if tied else host(dw.t()).T, r["dw"], bound)


# ---------------------------------------------------------------------------
# more than 2^32 bytes and values
# ---------------------------------------------------------------------------

def test_lookup_and_gradient_far_into_a_table(dev):
    from minitorch_amd import kernels as K

    V, C = (1 << 25) + 77, 132  # 4.4e9 values
    rng = np.random.default_rng(1)
    far = np.array([0, 5, V // 2, V - 2, V - 1])
    rows = rounded(rng.standard_normal((len(far), C)), "bfloat16")
    table = empty((V, C), "bfloat16")
    for i, v in enumerate(far):
        table[int(v):int(v) + 1].copy_(dev_array(rows[i:i + 1], "bfloat16"))
    at = rng.integers(0, len(far), 3000)
    ids = dev_array(far[at], "int64")
    assert np.array_equal(host(K.embedding_lookup(table, ids, scale=2.0)), rounded(2.0 * rows[at], "bfloat16"))
    del table
    dw = empty((V, C))  # 17.7 GB, of which the rows looked at are set
    for v in far:
        dw[int(v):int(v) + 1].copy_(np.ones((1, C), np.float32))
    for n in (1000, 3000):  # in one launch, and sorted
        g = rng.integers(-4, 5, (n, C)).astype(np.float32)  # sums are exact
        K.embedding_grad(dev_array(far[at[:n]], "int64"), dev_array(g), dw, accumulate=True)
        for i, v in enumerate(far):
            want = 1 + g[at[:n] == i].sum(0) if n == 1000 else before[i] + g[at[:n] == i].sum(0)
            assert np.array_equal(host(dw[int(v):int(v) + 1])[0], want)
        before = [host(dw[int(v):int(v) + 1])[0].copy() for v in far]


def test_dropout_of_more_than_32_bits_of_values(dev):
    from minitorch_amd import kernels as K

    rows, cols = (1 << 20) + 3, 4100
    x = full((rows, cols), 1.0, "bfloat16")
    y = K.dropout(x, 0.5, 3, 11, out=x)
    for r in (0, rows // 2, rows - 5):
        part = K.dropout(full((5, cols), 1.0, "bfloat16"), 0.5, 3, 11 + r * cols // 4)
        assert np.array_equal(host(y[r:r + 5]), host(part))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_xent_logits_of_more_than_32_bits_of_bytes(dev, dtype):
    """All logits at once (4.8 GB, and as much or more of their gradients) and 1024 rows
    at a time: each is off by at most its bounds, so they differ by at most twice those."""
    from minitorch_amd import kernels as K

    n, C, V = 40000, 16, 30011
    rng = np.random.default_rng(5)
    x = rounded(rng.uniform(-1, 1, (n, C)) * np.linspace(0.1, 4, n)[:, None], dtype)
    w = rounded(rng.uniform(-1, 1, (C, V)), dtype)
    labels = tokens(rng, n, V, 0.1)
    args = dev_array(x, dtype), dev_array(w, dtype), dev_array(labels, "int64")
    got = []
    for size in (1 << 33, 1024 * 30016 * 4):
        dx, dw = empty((n, C)), empty((C, V))
        loss, row, lse = K.linear_xent(*args, dx=dx, dw=dw, logits_bytes=size)
        got.append([host(t).copy() for t in (lse, row, dx)])
        assert np.isfinite(host(dw)).all()
    some = rng.choice(n, 60, replace=False)
    some[:4] = 0, 1, n - 2, n - 1
    r = ref.linear_xent(x[some], w, labels[some])
    bd = xent_bounds(x[some], w, None, r, dtype, "float32")
    count = ((labels >= 0) & (labels < V)).sum()
    mine = max(1, r["some"].sum())
    for lse, row, dx in got:
        inside(lse[some], r["lse"], bd[0])
        inside(row[some], r["row_loss"], bd[1])
        inside(dx[some], r["dx"] * mine / count, (bd[3] + 2 * U * np.abs(r["dx"])) * mine / count)
    assert np.abs(got[0][0] - got[1][0]).max() <= 2 * bd[0].max() and np.isfinite(got[0][2]).all()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def step_of(K, ids, labels, w, wt, x, y, dx, dw, db, b, dt, p, seed):
    """Lookup, dropout, projection with its loss, and the gradients back into the table."""
    K.embedding_lookup(w, ids, scale=2.0, out=x)
    K.dropout(x, p, seed, 0, out=y)
    loss, row, lse = K.linear_xent(y, wt, labels, bias=b, dx=dx, dw=dw, db=db)
    K.dropout(dx, p, seed, 0, out=dx)
    K.embedding_grad(ids, dx, dt, scale=2.0)
    return loss, row, lse


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,C,V", [(50, 24, 70), (4500, 32, 100), (5000, 16, 900)])
def test_a_recorded_step_is_the_eager_one(dev, n, C, V, dtype):
    """Two recorded steps over buffers of their own, replayed in turn with other tokens
    each time and eager calls between: every replay has the bits of the eager step."""
    from minitorch_amd import graphs
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(n)
    w = rounded(rng.standard_normal((V, C)), dtype)
    wd, b = dev_array(w, dtype), dev_array(rng.standard_normal(V))

    def memory():
        return dict(ids=dev_array(np.zeros(n), "int64"), labels=dev_array(np.zeros(n), "int64"), w=wd, wt=wd.t(),
                    x=empty((n, C), dtype), y=empty((n, C), dtype), dx=empty((n, C), dtype),
                    dw=empty((V, C), dtype).t(), db=empty((V,)), b=b, dt=empty((V, C)), p=0.3, seed=12)

    def values(m, outs):
        return [host(t).copy() for t in (*outs, m["x"], m["y"], m["dx"], m["dw"].t(), m["db"], m["dt"])]

    eager, sets = memory(), [memory(), memory()]
    step_of(K, **eager)
    recorded = []
    for m in sets:
        g = graphs.Graph()
        with g.capture():
            outs = step_of(K, **m)
        recorded.append((g, m, outs))
    for turn in range(3):
        for g, m, outs in recorded:
            ids, labels = tokens(rng, n, V), tokens(rng, n, V)
            for t in (eager, m):
                t["ids"].copy_(ids)
                t["labels"].copy_(labels)
            want = values(eager, step_of(K, **eager))
            g.replay()
            K.embedding_grad(eager["ids"], eager["dx"], empty((V, C)))  # eager work behind the replay
            assert all(np.array_equal(a, c, equal_nan=True) for a, c in zip(want, values(m, outs)))
            assert np.isfinite(want[0]).all()
        # the whole against float64, from the values the step itself stored
        keep = ref.keep((n, C), 0.3, 12)
        inside(want[3], ref.lookup(w, ids, 2.0), (U if dtype == "float32" else B) * np.abs(ref.lookup(w, ids, 2.0)))
        y = rounded(np.where(keep, want[3] * np.float32(1 / 0.7), np.float32(0)), dtype)
        assert np.array_equal(want[4], y)
        r = ref.linear_xent(y, w.T, labels, host(b))
        bd = xent_bounds(y, w.T, host(b), r, dtype, dtype)
        inside(want[2], r["lse"], bd[0])
        inside(want[6], r["dw"].T, bd[4].T)
        gx = np.where(keep, r["dx"] / 0.7, 0)
        got = want[5]
        inside(got, gx, np.where(keep, (bd[3] + (U if dtype == "float32" else B) * 2 * (np.abs(gx) + bd[3])) / 0.7, 0))
        dt, size = ref.lookup_grad(ids, got, V, 2.0)
        counts = np.bincount(ids[(ids >= 0) & (ids < V)], minlength=V)[:, None]
        inside(want[8], dt, (counts + 2) * U * size)
