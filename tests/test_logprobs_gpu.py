"""Token log probabilities, entropy, alternatives and their gradient on the GPU
against the plain float64 forms (oracle.paged.logprobs, logprobs_grad).

Bounds, with u = 2^-24: a term exp(x - max) is off by 2 u (|x| + |max|) + 4 u
relative (the scaling, the difference, the exponential) and a row's sum, added
in chains of at most V / 64 + 64 terms, by that many u more: e in all.  lse and
log probabilities are off by e + 4 u of their own magnitudes, the entropy by e
times its terms p (1 + |log p|), a probability by 2 e relative."""
import numpy as np
import pytest
from devarrays import H as host, T as dev_array, empty, full

from oracle import paged as ref
from oracle.attention import bf16_round

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(rng, rows, V, dtype, std=3.0):
    x = (std * rng.standard_normal((rows, V))).astype(np.float32)
    tokens = rng.integers(0, V, rows)
    tokens[::3] = x.argmax(1)[::3]
    return (bf16_round(x) if dtype == "bfloat16" else x), tokens.astype(np.int64)


def bounds(x, scale, r):
    """(log probability, entropy, lse, probability-relative) bounds per row."""
    V = x.shape[1]
    finite = np.where(np.isfinite(x), np.abs(x), 0.0) * scale
    mag = finite.max(1)
    lse = np.where(np.isfinite(r[2]), np.abs(r[2]), 0.0)
    e = U * (4 * mag + V / 64 + 64 + 8)
    p = r[5]
    with np.errstate(divide="ignore", invalid="ignore"):
        terms = np.where(p > 0, p * (1 + np.abs(np.log(p))), 0.0).sum(1)
    return e + 4 * U * (lse + mag), 3 * e * terms + 8 * U, e + 4 * U * (lse + mag), 3 * e + 4 * U * (lse + mag)


def grad_bound(x, tokens, scale, r, g, gh, want):
    """Bound of the gradient's entries, from those of the probabilities."""
    V, pb = x.shape[1], bounds(x, scale, r)[3]
    with np.errstate(invalid="ignore", divide="ignore"):
        lp = np.where(r[5] > 0, np.abs(np.log(r[5])), 0.0)
    size = np.abs(g)[:, None] + np.abs(gh)[:, None] * (lp + np.abs(r[1])[:, None] + 1)
    own = np.where(np.arange(V) == tokens[:, None], np.abs(g)[:, None], 0.0)
    return scale * r[5] * size * (pb + 8 * U)[:, None] + 4 * U * np.abs(want) + 4 * U * scale * own + 1e-30


def check(x, tokens, dtype, scale=1.0, top=0, grad=True, ld=0, seed=0):
    """Forward and gradient of one call; ld: values between rows' ends."""
    from minitorch_amd import kernels as K

    rows, V = x.shape
    wide = np.full((rows, V + ld), np.nan, np.float32)
    wide[:, :V] = x
    dx = dev_array(wide, dtype)[:, :V]
    dt = dev_array(tokens, "int64")
    out = K.token_logprobs(dx, dt, top=top, scale=scale)
    r = ref.logprobs(x, tokens, scale, top)
    lb, eb, sb, _ = bounds(x, scale, r)
    got = [host(t) for t in out]
    assert np.array_equal(got[3], r[3])
    for g, want, b in ((got[0], r[0], lb), (got[1], r[1], eb), (got[2], r[2], sb), (got[4], r[4], lb[:, None])):
        same = (g == want) | (np.isnan(g) & np.isnan(want))
        with np.errstate(invalid="ignore"):
            assert np.all(same | (np.abs(g - want) <= b)), float(np.nanmax(np.abs(g - want) / b))
    if not grad:
        return got
    rng = np.random.default_rng(seed)
    g, gh = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    want = ref.logprobs_grad(x, tokens, g, gh, scale)
    bound = grad_bound(x, tokens, scale, r, g, gh, want)
    old = rng.standard_normal((rows, V + ld)).astype(np.float32)
    for acc in (False, True):
        buf = dev_array(old)
        K.token_logprobs_bwd(dx, dt, out[2], out[1], dev_array(g), dev_array(gh), scale=scale, dlogits=buf[:, :V],
                             accumulate=acc)
        d = host(buf)
        assert np.array_equal(d[:, V:], old[:, V:])
        target = want + (old[:, :V] if acc else 0)
        assert np.all(np.abs(d[:, :V] - target) <= bound + (2 * U * (np.abs(old[:, :V]) + np.abs(want)) if acc else 0))
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [1, 2, 3, 15, 17, 48, 49, 63, 64, 65, 80, 81, 128, 129, 255, 256, 257, 511, 512, 513, 1000,
                               1023, 1024, 1025, 2047, 2049, 4095, 4097, 5003, 8192, 8193])
def test_vocabulary_sizes(dev, dtype, V):
    rng = np.random.default_rng(V)
    x, tok = make(rng, 9, V, dtype)
    check(x, tok, dtype, top=min(5, V), ld=V % 4)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,V", [(1, 50021), (3, 131072), (40, 20000), (300, 8193), (257, 32768), (256, 40000)])
def test_large_vocabularies(dev, dtype, rows, V):
    rng = np.random.default_rng(rows)
    x, tok = make(rng, rows, V, dtype)
    check(x, tok, dtype, scale=1.25, top=20)


@pytest.mark.parametrize("rows", [1, 2, 255, 257, 1031, 70001])
def test_rows(dev, rows):
    rng = np.random.default_rng(rows)
    x, tok = make(rng, rows, 33, "float32")
    check(x, tok, "float32", scale=0.7, top=3)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V,top", [(1, 1), (7, 7), (64, 64), (100, 64), (900, 33), (5000, 64), (40000, 64)])
def test_alternatives(dev, dtype, V, top):
    rng = np.random.default_rng(top)
    x, tok = make(rng, 5, V, dtype)
    check(x, tok, dtype, top=top, grad=False)


@pytest.mark.parametrize("V,ld", [(1, 0), (2, 1), (5, 0), (63, 0), (1025, 0), (8195, 0), (8196, 1), (20001, 0),
                                  (50021, 0)])
def test_rows_at_odd_addresses(dev, V, ld):
    """bf16 rows of which every other begins between two words: their first and
    last values the largest, equal to others, hidden and alone."""
    rng = np.random.default_rng(V)
    x, tok = make(rng, 12, V, "bfloat16")
    x[0:2, 0] = 30.0
    x[2:4, [0, V // 2, V - 1]] = 25.0
    x[4:6, 0] = -np.inf
    x[6:8, 1:] = -np.inf
    x[8:10, :-1] = -np.inf
    tok[::3] = 0
    tok[1::3] = V - 1
    if V < 3:  # no row without any
        x[4:10] = 1.0
    check(x, tok, "bfloat16", top=min(V, 5), ld=ld)


@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "two_values", "blocks", "signed_zero"])
@pytest.mark.parametrize("V", [65, 700, 33333])
def test_alternatives_of_ties_and_orders(dev, kind, V):
    """Ties go to the lowest id, whatever the order of the row."""
    i = np.arange(V)
    x = {"equal": 0 * i, "ascending": i / V, "descending": -i / V, "two_values": i % 2, "blocks": (i // 64) % 5,
         "signed_zero": np.where(i % 3 == 0, -0.0, 0.0)}[kind].astype(np.float32)
    x = np.stack([x, x[::-1]])
    check(x, np.array([0, V - 1]), "float32", top=min(V, 40), grad=kind == "equal")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [50, 3000, 30001])
def test_hidden_logits_and_rows_of_nothing(dev, dtype, V):
    """-inf logits have probability 0, also the given token's; a row of nothing
    else has no distribution; tokens outside the vocabulary are no tokens."""
    rng = np.random.default_rng(3)
    x, tok = make(rng, 8, V, dtype)
    x[0, rng.random(V) < 0.5] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, V // 2] = 1.0  # certain
    x[3, tok[3]] = -np.inf
    x[4, 1:] = -np.inf
    tok[4] = V - 1
    tok[5], tok[6], tok[7] = -1, V, -(2 ** 40)
    check(x, tok, dtype, top=6)


def test_not_a_number_and_infinity(dev):
    """NaN anywhere, or +inf, makes a row's numbers NaN; its alternatives are
    still in order, NaN first.  Other rows are not touched."""
    rng = np.random.default_rng(4)
    x, tok = make(rng, 4, 600, "float32")
    x[1, 5], x[1, 300] = np.nan, -np.nan
    x[2, 17] = np.inf
    got = check(x, tok, "float32", top=4, grad=False)
    assert np.isnan(got[2][1:3]).all() and np.isfinite(got[2][[0, 3]]).all()


def test_wide_ranges(dev):
    """Logits of +-1e4 neither overflow nor lose the entropy of near certainty."""
    rng = np.random.default_rng(5)
    x, tok = make(rng, 6, 2000, "float32", std=3e3)
    check(x, tok, "float32", top=3)
    x = np.zeros((2, 4), np.float32)
    x[0, 0], x[1] = 15.0, [0, -20, -30, 3]
    got = check(x, np.array([0, 1]), "float32")
    # l = 1 + 9e-7 is rounded once, what the entropy is made of is not lost
    want = ref.logprobs(x, np.array([0, 1]))[1]
    assert np.all(np.abs(got[1] - want) <= 4 * U + 64 * U * want)


def test_gradient_against_differences(dev):
    """The gradient of sum(g logprob + gh entropy) against central differences
    of the float64 form: step h, error h^2 / 6 times a third derivative of at
    most 24 scale^3 (|g| + |gh| (2 + max |log p|)), plus its rounding and the
    fp32 gradient's own 128 u of scale times that size."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(6)
    rows, V, scale, h = 2, 11, 1.3, 1e-4
    x, tok = make(rng, rows, V, "float32", std=1.0)
    g, gh = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    dx, dt = dev_array(x), dev_array(tok, "int64")
    lp, ent, lse, _, _ = K.token_logprobs(dx, dt, scale=scale)
    d = host(K.token_logprobs_bwd(dx, dt, lse, ent, dev_array(g), dev_array(gh), scale=scale))

    def f(y):
        r = ref.logprobs(y, tok, scale)
        return g @ r[0] + gh @ r[1]

    size = np.abs(g).max() + np.abs(gh).max() * (2 + np.abs(np.log(ref.logprobs(x, tok, scale)[5])).max())
    for r in range(rows):
        for v in range(V):
            a, b = x.astype(np.float64), x.astype(np.float64)
            a[r, v] += h
            b[r, v] -= h
            assert abs((f(a) - f(b)) / (2 * h) - d[r, v]) <= 4 * h * h * size * scale ** 3 + 1e-15 / h * 100 + 128 * U * scale * size


def test_gradient_of_one_output_alone(dev):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(7)
    x, tok = make(rng, 5, 130, "float32")
    dx, dt = dev_array(x), dev_array(tok, "int64")
    _, ent, lse, _, _ = K.token_logprobs(dx, dt)
    g = rng.standard_normal(5).astype(np.float32)
    z = np.zeros(5, np.float32)
    for a, b in ((g, None), (None, g), (None, None)):
        d = host(K.token_logprobs_bwd(dx, dt, lse, ent, None if a is None else dev_array(a),
                                      None if b is None else dev_array(b)))
        a, b = z if a is None else a, z if b is None else b
        want = ref.logprobs_grad(x, tok, a, b)
        assert np.all(np.abs(d - want) <= grad_bound(x, tok, 1.0, ref.logprobs(x, tok), a, b, want))


def test_recorded_calls(dev):
    """Two recorded calls of different sizes replayed in turn with eager work
    between, on rows that change: the eager results, bit for bit."""
    from minitorch_amd import kernels as K
    from minitorch_amd.graphs import Graph

    rng = np.random.default_rng(8)
    sets = []
    for rows, V, top in ((4, 40000, 10), (50, 300, 5)):
        s = dict(x=empty((rows, V)), t=full((rows,), 0, "int64"), shape=(rows, V))
        s["x"].fill_(0.0)

        def call(s=s, top=top):
            return K.token_logprobs(s["x"], s["t"], top=top)

        call()
        s["call"], s["graph"] = call, Graph()
        with s["graph"].capture():
            s["out"] = call()
        sets.append(s)
    for _ in range(4):
        for s in sets:
            x, tok = make(rng, *s["shape"], "float32")
            s["x"].copy_(x)
            s["t"].copy_(tok)
            want = [host(t) for t in s["call"]()]
            s["graph"].replay()
            assert all(np.array_equal(host(a), b) for a, b in zip(s["out"], want))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [7, 65, 300, 700, 5003, 50021])
@pytest.mark.parametrize("scale", [2.0 ** -89, 1e-20, 1e20, 1e37])
def test_scales_at_the_ends(dev, dtype, V, scale):
    """Scales near the ends of what is taken, with hidden logits: a nearly
    even distribution over the others, or one value."""
    rng = np.random.default_rng(V)
    x, tok = make(rng, 6, V, dtype)
    x[1, ::2] = -np.inf
    x[2, 1:] = -np.inf
    x[3, 1::2] = np.finfo(np.float32).min if dtype == "float32" else -3e38
    tok[1:4] = 0
    x *= np.float32(0.1) if scale > 1 else np.float32(1)
    if dtype == "bfloat16":
        x = bf16_round(x)
    from minitorch_amd import kernels as K

    lp, ent, lse, _, _ = (host(t) for t in K.token_logprobs(dev_array(x, dtype), dev_array(tok, "int64"), scale=scale))
    xd = x.astype(np.float64) * scale
    d = xd - xd.max(1, keepdims=True)
    logl = np.log(np.exp(d).sum(1))
    p = np.exp(d - logl[:, None])
    want = np.take_along_axis(d, tok[:, None], 1)[:, 0] - logl
    e = U * (V / 64 + 80)
    # differences are formed before the scale: 3 u of them
    with np.errstate(invalid="ignore"):
        assert np.all((lp == want) | (np.abs(lp - want) <= e + 4 * U * (np.abs(want) + logl)))
    ld = np.log(np.where(p > 0, p, 1))
    terms = (p * (1 + np.abs(ld))).sum(1)
    # an exponent d scale is off by 3 u of itself, so is what its term adds
    assert np.all(np.abs(ent + (p * ld).sum(1)) <= 3 * e * terms + 8 * U * (1 + logl) + 4 * U * (p * ld ** 2).sum(1))
    if scale <= 1:
        assert np.all(np.abs(lse - (xd.max(1) + logl)) <= e + 4 * U * (logl + np.abs(xd.max(1))))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("gradient", [1e9, -1e12, 1e30])
def test_gradient_of_large_upstream_gradients_at_hidden_logits(dev, dtype, gradient):
    """-inf, the type's lowest value and logits far below the others get 0
    whatever comes from upstream; the others the formula's."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(5)
    x, tok = make(rng, 4, 130, dtype)
    low = np.float32(np.finfo(np.float32).min) if dtype == "float32" else np.float32(-3.3e38)
    x[:, 3], x[:, 50], x[:, 70] = -np.inf, low, -500.0
    if dtype == "bfloat16":
        x = bf16_round(x)
    tok[:] = 1
    dx, dt = dev_array(x, dtype), dev_array(tok, "int64")
    _, ent, lse, _, _ = K.token_logprobs(dx, dt)
    g = np.full(4, gradient, np.float32)
    d = host(K.token_logprobs_bwd(dx, dt, lse, ent, None, dev_array(g)))
    assert not d[:, [3, 50, 70]].any()
    seen, none = [i for i in range(130) if i not in (3, 50, 70)], np.zeros(4, np.float32)
    x, d = x[:, seen], d[:, seen]
    want = ref.logprobs_grad(x, tok, none, g)
    assert np.all(np.abs(d - want) <= grad_bound(x, tok, 1.0, ref.logprobs(x, tok), none, g, want))
