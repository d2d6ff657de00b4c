"""The paged key-value cache on the GPU against its plain float64 forms
(oracle.paged): append, one-token attention with the weights rows receive, and
eviction, each alone and in a decoding loop.

Bounds, with u = 2^-24 (half a step of fp32): a score is a D-term fp32 dot
product times the scale, off by at most E = (D + 8) u scale max_j sum|q k_j|; a
weight exp(s - lse) is then off by 2 E + (n + 32) u relative (numerator and the
n-term denominator), plus 2^-16 over bf16 pools, where weights enter the matrix
products as two bf16 pieces (fp32 rows: three, 2^-23); an output adds the same
relative error of sum p|v|, the n u of its own sum and, in bf16, half a step
2^-8 of its value."""
import numpy as np
import pytest
from devarrays import H as host, T as dev_array, empty, full

from oracle import paged as ref
from oracle.attention import bf16_round

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16")]


def rounded(x, dtype):
    return bf16_round(x) if dtype == "bfloat16" else x.astype(np.float32)


def make_table(rng, lengths, page, spare=0):
    """A table over shuffled pages (-1 behind a sequence's), pages in all and
    the ids no table uses."""
    need = [-(-n // page) for n in lengths]
    total = max(1, sum(need) + spare)
    ids = rng.permutation(total).astype(np.int32)
    table = np.full((len(lengths), max(1, max(need))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, total, ids[at:]


def make_pool(rng, n, h, page, d, dtype):
    return rounded(rng.standard_normal((n, h, page, d), dtype=np.float32), dtype)


def to_device(pool, dtype, layout):
    """The pool as a (n, heads, page, D) view, stored by heads or by rows."""
    if layout == "rows":
        return dev_array(pool.transpose(0, 2, 1, 3), dtype).transpose(1, 2)
    return dev_array(pool, dtype)


def host_pool(pool):
    """Host copy of a pool view (16-bit copies need contiguous memory)."""
    return host(pool) if pool.is_contiguous() else host(pool.transpose(1, 2)).transpose(0, 2, 1, 3)


def decode_bounds(case, r, n):
    """(o, lse, weight-per-head) bounds of a ref.decode result."""
    o, lse, w, qk, pv = r
    D = o.shape[-1]
    E = (D + 8) * U * qk
    split = {"float32": 0.0, "bfloat16": 2.0 ** -16}[case["q"]] if case["cache"] == "bfloat16" else 0.0
    if case["cache"] == "bfloat16" and case["q"] == "float32":
        split = 2.0 ** -22
    rel = 2 * E + (n + 32) * U
    ob = pv * (rel + split + (n + 32) * U)[..., None, None]
    ob = ob + np.abs(o) * (2.0 ** -8 if case["q"] == "bfloat16" else 2 * U) + 1e-30
    lb = E + (n + 32) * U + 4 * U * np.abs(np.where(np.isfinite(lse), lse, 0.0))
    return ob, lb, rel


def check_decode(case, lengths, seed, edit=None, in_place=False, with_lse=True):
    """One call against the oracle; `edit` may change the host arrays."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(seed)
    B, H, Hkv, D, page = len(lengths), case["H"], case["Hkv"], case["D"], case["page"]
    table, total, _ = make_table(rng, lengths, page, spare=1)
    kp, vp = (make_pool(rng, total, Hkv, page, D, case["cache"]) for _ in range(2))
    q = rounded(2 * rng.standard_normal((B, H, 1, D), dtype=np.float32), case["q"])
    cap = table.shape[1] * page
    w_in = rng.random((B, Hkv, cap + 3), dtype=np.float32)
    a = dict(q=q, kp=kp, vp=vp, table=table, lengths=np.array(lengths, np.int32), w_in=w_in)
    if edit is not None:
        edit(a, rng)
    q, kp, vp, table, lens, w_in = (a[k] for k in ("q", "kp", "vp", "table", "lengths", "w_in"))
    scale = 1.0 / np.sqrt(D)
    dk, dv = (to_device(p, case["cache"], case.get("layout", "heads")) for p in (kp, vp))
    lse = full((B, H), 7.0) if with_lse else None
    kw = {}
    if case.get("weights"):
        win = dev_array(w_in)
        wout = win if in_place else full(w_in.shape, -5.0)
        kw = dict(weights=wout, weights_in=win)
    o, _ = K.attn_decode_paged(dev_array(q, case["q"]), dk, dv, dev_array(table, "int32"),
                               dev_array(lens, "int32"), scale, lse=lse, **kw)
    r = ref.decode(q, kp, vp, table, lens, scale)
    n = int(max(1, min(cap, max(lens))))
    ob, lb, rel = decode_bounds(case, r, n)
    got = host(o).astype(np.float64)
    assert np.all(np.abs(got - r[0]) <= ob), float((np.abs(got - r[0]) / ob).max())
    if with_lse:
        got = host(lse).astype(np.float64)
        empty_rows = np.isneginf(r[1])
        assert np.array_equal(np.isneginf(got), empty_rows)
        some = ~empty_rows
        assert np.all(np.abs(got[some] - r[1][some]) <= lb[some])
    if case.get("weights"):
        got = host(wout).astype(np.float64)
        want = w_in.astype(np.float64)
        want[..., :cap] += r[2]
        G = H // Hkv
        relw = rel.reshape(B, Hkv, G).max(-1)[..., None]
        seen = np.arange(cap + 3) < np.clip(lens, 0, cap)[:, None, None]
        seen = np.broadcast_to(seen, got.shape)
        bound = np.zeros_like(want)
        bound[..., :cap] = r[2] * relw
        bound += (G + 2) * U * np.abs(want) + 1e-30
        assert np.all(np.abs(got - want)[seen] <= bound[seen])
        behind = w_in if in_place else np.full_like(w_in, -5.0)
        assert np.array_equal(host(wout)[~seen], behind[~seen])
    # nothing is written to the pool
    assert np.array_equal(host_pool(dk), kp, equal_nan=True) and np.array_equal(host_pool(dv), vp, equal_nan=True)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("page,layout", [(16, "heads"), (16, "rows"), (7, "rows"), (64, "heads"), (1, "heads")])
def test_decode_types_sizes_and_layouts(dev, q, cache, D, page, layout):
    case = dict(q=q, cache=cache, H=6, Hkv=3, D=D, page=page, layout=layout, weights=True)
    check_decode(case, [1, page, page + 1, 33, 97, 0, 256], seed=D + page)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 1), (16, 1), (17, 1), (40, 2), (12, 4)])
def test_decode_head_groups(dev, q, cache, H, Hkv):
    case = dict(q=q, cache=cache, H=H, Hkv=Hkv, D=64, page=16, weights=True)
    check_decode(case, [5, 160, 48], seed=H)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("lengths", [[1], [2], [31], [32], [33], [1000, 17], [4097], [2049, 1, 2048]])
@pytest.mark.parametrize("weights", [False, True])
def test_decode_lengths(dev, q, cache, lengths, weights):
    case = dict(q=q, cache=cache, H=2, Hkv=1, D=64, page=32, weights=weights)
    check_decode(case, lengths, seed=sum(lengths), with_lse=not weights, in_place=weights)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("page", [2, 4, 12, 20, 48])
def test_decode_page_sizes(dev, q, cache, page):
    """Pages that hold whole runs of 16 rows, of 4, and neither."""
    case = dict(q=q, cache=cache, H=3, Hkv=1, D=32, page=page, layout="rows", weights=True)
    check_decode(case, [1, 3 * page - 1, 130, 0, 257], seed=page)


@pytest.mark.parametrize("page", [4, 16])
def test_decode_rows_far_apart(dev, page):
    """Row strides that 32-bit offsets from a page do not reach."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(page)
    n, D, far = 3, 16, 1 << 24
    pools = [rng.standard_normal((n, 1, page, D), dtype=np.float32) for _ in range(2)]
    base = empty(((page - 1) * far + n * D,), "float32")
    views = []
    for i, pool in enumerate(pools):  # page p's rows at p D, one `far` apart; V half a stride on
        view = base.as_strided((n, 1, page, D), (D, D, far, 1), 0)
        if i:
            base = empty(((page - 1) * far + n * D,), "float32")
            view = base.as_strided((n, 1, page, D), (D, D, far, 1), 0)
        for r in range(page):
            view[:, :, r].copy_(dev_array(pool[:, :, r]))
        views.append(view)
    table, lens = np.array([[2, 0, 1]], np.int32), np.array([3 * page - 1], np.int32)
    q = rng.standard_normal((1, 2, 1, D), dtype=np.float32)
    o, _ = K.attn_decode_paged(dev_array(q), *views, dev_array(table, "int32"), dev_array(lens, "int32"), 0.25)
    r = ref.decode(q, *pools, table, lens, 0.25)
    ob, _, _ = decode_bounds(dict(q="float32", cache="float32"), r, 3 * page)
    assert np.all(np.abs(host(o) - r[0]) <= ob)


@pytest.mark.parametrize("B,H,Hkv,D,lengths", [
    (1, 2, 1, 16, (512, 513)), (130, 1, 1, 16, (1000, 1024, 700)), (100, 8, 8, 16, (2000, 60, 1100)),
    (1, 20, 1, 32, (1500,)), (2, 34, 2, 16, (3000, 1)), (9, 17, 1, 16, (1300, 5))])
@pytest.mark.parametrize("weights", [False, True])
def test_decode_one_chunk_and_many(dev, B, H, Hkv, D, lengths, weights):
    """Around the sizes where a sequence takes one workgroup, or several that
    a second launch joins, with more than 16 heads a K/V head too."""
    for n in ([lengths] if B > 1 else [(x,) for x in lengths]):
        case = dict(q="bfloat16", cache="bfloat16", H=H, Hkv=Hkv, D=D, page=16, weights=weights)
        check_decode(case, [n[i % len(n)] for i in range(B)], seed=B + n[0])


@pytest.mark.parametrize("page,D", [(32, 128), (37, 64)])
def test_decode_long_cache(dev, page, D):
    case = dict(q="bfloat16", cache="bfloat16", H=4, Hkv=1, D=D, page=page, weights=True)
    check_decode(case, [40001], seed=3)


@pytest.mark.parametrize("H,Hkv,D,page,lengths", [
    (4, 2, 128, 64, [20000, 300, 1, 300, 300]),
    (2, 1, 64, 16, [0, 5000, 0, 0, 63, 64, 65, 8001, 256, 0]),
    (8, 4, 64, 16, [2304] * 4),
    (8, 4, 64, 16, [2304, 4608]),
    (1, 1, 16, 8, [1 + 37 * i % 4000 for i in range(128)]),
    (1, 1, 16, 16, [4000] + [0] * 126 + [1]),
    (2, 1, 16, 1, [9000, 100, 4033, 4032]),
    (64, 2, 32, 20, [3000, 1000, 2999]),
    (2048, 8, 16, 16, [2500]),
    (12, 12, 16, 32, [6000, 700]),
    (48, 1, 64, 64, [9000, 3000]),
    (96, 2, 16, 16, [2200 + 9 * i for i in range(40)]),
    (1, 1, 16, 16, [1 + 41 * i % 2500 for i in range(130)]),
    (9, 9, 16, 16, [8100 - 517 * i for i in range(15)]),
    (3, 3, 16, 16, [4096 - 30 * i for i in range(128)])],
    ids=["skewed", "empty_between", "equal", "twice", "128_sequences", "first_and_last", "pages_of_one", "head_tiles",
         "many_head_tiles", "more_heads", "three_head_tiles", "80_of_three", "130_sequences", "chunks_of_8", "whole_of_4096"])
@pytest.mark.parametrize("weights", [False, True])
def test_decode_cuts(dev, H, Hkv, D, page, lengths, weights):
    """How sequences are shared out among workgroups: by the lengths of all, in
    chunks alike, and whole."""
    case = dict(q="bfloat16", cache="bfloat16", H=H, Hkv=Hkv, D=D, page=page, weights=weights)
    check_decode(case, lengths, seed=len(lengths) + H)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("H,Hkv,D,lengths", [
    (8, 4, 16, [1 + 11 * i % 700 for i in range(70)]),
    (34, 2, 16, [1 + 11 * i % 300 for i in range(64)]),
    (4, 4, 16, [3000, 100, 0, 5000]),
    (40, 2, 32, [2900, 1400]),
    (4, 4, 16, [2500 - 60 * i for i in range(40)]),
    (5, 5, 32, [9000, 1])])
def test_decode_heads_that_share_lines(dev, q, cache, H, Hkv, D, lengths):
    case = dict(q=q, cache=cache, H=H, Hkv=Hkv, D=D, page=16, layout="rows", weights=H == 8)
    check_decode(case, lengths, seed=H + D)


def test_decode_nothing_cached(dev):
    """A wide table and no rows at all: zeros and -inf, weights as they were."""
    def edit(a, rng):
        a["lengths"] = np.array([0, 0, -1], np.int32)

    case = dict(q="float32", cache="float32", H=4, Hkv=2, D=64, page=16, weights=True)
    check_decode(case, [3000, 20, 700], seed=2, edit=edit)


def test_decode_lengths_behind_the_table_and_negative(dev):
    def edit(a, rng):
        a["lengths"] = np.array([10 ** 9, -4, 20], np.int32)

    case = dict(q="float32", cache="float32", H=2, Hkv=2, D=32, page=8, weights=True)
    check_decode(case, [24, 24, 24], seed=9, edit=edit)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("page", [16, 5])
def test_decode_rows_that_are_not_there(dev, q, cache, page):
    """Page ids outside the pool are holes, in the middle, at the ends, and
    over whole sequences."""
    def edit(a, rng):
        t, n = a["table"], a["kp"].shape[0]
        t[0, 1] = -1
        t[1, 0] = n
        t[1, -1] = 2 ** 31 - 1
        t[2, :] = -2 ** 31
        t[3, 2:] = -7

    case = dict(q=q, cache=cache, H=4, Hkv=2, D=64, page=page, weights=True)
    check_decode(case, [6 * page] * 4, seed=page, edit=edit)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("page", [16, 6])
def test_decode_does_not_see_what_lies_behind(dev, q, cache, page):
    """NaN and infinities in rows behind the last and in unused pages."""
    lengths = [1, page - 1, 2 * page + 1, 50]

    def edit(a, rng):
        n = a["kp"].shape[0]
        used = np.zeros((n, page), bool)
        for b, m in enumerate(lengths):
            for j in range(m):
                used[a["table"][b, j // page], j % page] = True
        for pool, bad in ((a["kp"], np.nan), (a["vp"], np.inf)):
            pool.transpose(0, 2, 1, 3)[~used] = bad

    case = dict(q=q, cache=cache, H=2, Hkv=2, D=32, page=page, weights=True)
    check_decode(case, lengths, seed=5, edit=edit)


def test_decode_shared_pages(dev):
    """Sequences that share a prompt's pages, and one that lists a page twice."""
    def edit(a, rng):
        a["table"][1, :3] = a["table"][0, :3]
        a["table"][2, 1] = a["table"][2, 0]

    case = dict(q="bfloat16", cache="bfloat16", H=8, Hkv=2, D=64, page=16, weights=True)
    check_decode(case, [70, 64, 40], seed=6, edit=edit)


def test_decode_large_scores(dev):
    """Scores up to some hundreds: nothing overflows, the largest wins."""
    def edit(a, rng):
        a["q"] = a["q"] * np.float32(16)

    case = dict(q="float32", cache="float32", H=3, Hkv=3, D=64, page=16, weights=True)
    check_decode(case, [100, 300], seed=7, edit=edit)


def test_decode_nan_that_is_seen(dev):
    """A NaN key row that is seen makes its head's output NaN, no other's."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(0)
    kp, vp = (make_pool(rng, 4, 2, 16, 64, "bfloat16") for _ in range(2))
    kp[1, 0, 3, 5] = np.nan
    q = rounded(rng.standard_normal((1, 2, 1, 64), dtype=np.float32), "bfloat16")
    o, _ = K.attn_decode_paged(dev_array(q, "bfloat16"), dev_array(kp, "bfloat16"), dev_array(vp, "bfloat16"),
                               dev_array(np.arange(4, dtype=np.int32)[None], "int32"),
                               dev_array(np.array([60], np.int32), "int32"), 0.125)
    o = host(o)
    assert np.isnan(o[0, 0]).all() and np.isfinite(o[0, 1]).all()


def test_decode_strided_operands(dev):
    """q and the output as views of packed tensors, the table as columns of a
    wider one, an expanded table row."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(2)
    B, H, D, page = 3, 4, 32, 8
    kp, vp = (make_pool(rng, 10, H, page, D, "float32") for _ in range(2))
    packed = rng.standard_normal((B, 1, 3, H, D), dtype=np.float32)
    wide = rng.integers(0, 10, (B, 7)).astype(np.int32)
    lens = np.array([40, 3, 25], np.int32)
    qd = dev_array(packed)[:, :, 1].transpose(1, 2)
    buf = full((B, 1, 2 * H, D), 9.0)
    out = buf[:, :, ::2].transpose(1, 2)
    td = dev_array(wide, "int32")[:, 1:6]
    args = (dev_array(kp), dev_array(vp), td, dev_array(lens, "int32"), 0.2)
    K.attn_decode_paged(qd, *args, out=out)
    q = packed[:, 0, 1][:, :, None]
    case = dict(q="float32", cache="float32")
    r = ref.decode(q, kp, vp, wide[:, 1:6], lens, 0.2)
    ob, _, _ = decode_bounds(case, r, 40)
    got = host(buf)
    assert np.all(np.abs(got[:, 0, ::2] - r[0][:, :, 0]) <= ob[:, :, 0])
    assert np.all(got[:, 0, 1::2] == 9.0)
    one = dev_array(wide, "int32")[:1, 1:6].expand(B, 5)
    o, _ = K.attn_decode_paged(qd, args[0], args[1], one, args[3], 0.2)
    r = ref.decode(q, kp, vp, np.repeat(wide[:1, 1:6], B, 0), lens, 0.2)
    assert np.all(np.abs(host(o) - r[0]) <= decode_bounds(case, r, 40)[0])


def test_decode_same_bits_every_time(dev):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(4)
    lens = [5000, 77]
    table, total, _ = make_table(rng, lens, 16)
    kp, vp = (dev_array(make_pool(rng, total, 2, 16, 64, "bfloat16"), "bfloat16") for _ in range(2))
    q = dev_array(rng.standard_normal((2, 8, 1, 64), dtype=np.float32), "bfloat16")
    t, ln = dev_array(table, "int32"), dev_array(np.array(lens, np.int32), "int32")
    first = None
    for _ in range(4):
        w = full((2, 2, table.shape[1] * 16), 0.0)
        lse = empty((2, 8))
        o, _ = K.attn_decode_paged(q, kp, vp, t, ln, 0.125, lse=lse, weights=w)
        got = [host(x) for x in (o, lse, w)]
        first = first or got
        assert all(np.array_equal(a, b) for a, b in zip(got, first))


def test_offsets_past_32_bits(dev):
    """A pool of more than 2^32 elements: its last pages are read, appended to
    and evicted into."""
    from minitorch_amd import device, kernels as K

    rng = np.random.default_rng(8)
    page, Hkv, D = 64, 8, 128
    n = (1 << 32) // (page * Hkv * D) + 5
    kd, vd = (empty((n, Hkv, page, D), "bfloat16") for _ in range(2))
    small = {}
    for name, pool in (("k", kd), ("v", vd)):
        small[name] = make_pool(rng, 3, Hkv, page, D, "bfloat16")
        pool[n - 3:].copy_(dev_array(small[name], "bfloat16"))
    new = rounded(rng.standard_normal((1, Hkv, 1, D), dtype=np.float32), "bfloat16")
    table = np.array([[n - 1, n - 3]], np.int32)
    local = np.array([[2, 0]], np.int32)
    lens = np.array([100], np.int32)
    td, ld = dev_array(table, "int32"), dev_array(lens, "int32")
    nd = dev_array(new, "bfloat16")
    K.kv_append_paged(nd, nd, kd, vd, td, ld)
    small = {k: ref.append(new, p, local, lens) for k, p in small.items()}
    q = rounded(rng.standard_normal((1, 16, 1, D), dtype=np.float32), "bfloat16")
    w = full((1, Hkv, 2 * page), 0.0)
    o, _ = K.attn_decode_paged(dev_array(q, "bfloat16"), kd, vd, td, ld, 0.1, weights=w)
    r = ref.decode(q, small["k"], small["v"], local, lens, 0.1)
    ob, _, _ = decode_bounds(dict(q="bfloat16", cache="bfloat16"), r, 100)
    assert np.all(np.abs(host(o) - r[0]) <= ob)
    wh = host(w)
    K.kv_evict_paged(kd, vd, td, ld, w, dev_array(np.array([[n - 2]], np.int32), "int32"), 50, 10)
    e = ref.evict(small["k"], small["v"], local, lens, wh, np.array([[1]], np.int32), 50, 10)
    assert np.array_equal(host(kd[n - 3:].clone()), e[0]) and np.array_equal(host(vd[n - 3:].clone()), e[1])
    del kd, vd
    device.empty_cache()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("D,page,layout", [(16, 16, "rows"), (64, 5, "heads"), (128, 1, "rows"), (32, 64, "heads")])
@pytest.mark.parametrize("T", [1, 3, 70])
def test_append(dev, rows, cache, D, page, layout, T):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(T + D)
    B, Hkv = 4, 3
    past = [0, 1, page, 2 * page + 3]
    counts = np.array([T, max(0, T - 1), 0, T // 2 + 1], np.int32)
    for cts in (None, counts):
        n = np.full(B, T) if cts is None else cts
        lens = (np.array(past) + n).astype(np.int32)
        table, total, _ = make_table(rng, [int(x) for x in lens], page, spare=2)
        kp, vp = (make_pool(rng, total, Hkv, page, D, cache) for _ in range(2))
        k, v = (rounded(rng.standard_normal((B, Hkv, T, D), dtype=np.float32), rows) for _ in range(2))
        dk, dv = (to_device(p, cache, layout) for p in (kp, vp))
        # new rows as a projection leaves them: (B, T, heads, D) read by heads
        xk, xv = (dev_array(x.transpose(0, 2, 1, 3), rows).transpose(1, 2) for x in (k, v))
        K.kv_append_paged(xk, xv, dk, dv, dev_array(table, "int32"), dev_array(lens, "int32"),
                          counts=None if cts is None else dev_array(cts, "int32"))
        assert np.array_equal(host_pool(dk), ref.append(rounded(k, cache), kp, table, lens, cts))
        assert np.array_equal(host_pool(dv), ref.append(rounded(v, cache), vp, table, lens, cts))


def test_append_rows_that_have_no_place(dev):
    """Rows before the first, behind the table and in pages outside the pool
    are skipped; counts above T count as T."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(1)
    page, D, T = 4, 16, 6
    kp, vp = (make_pool(rng, 6, 1, page, D, "float32") for _ in range(2))
    k, v = (rng.standard_normal((4, 1, T, D), dtype=np.float32) for _ in range(2))
    table = np.array([[0, 1], [2, -1], [6, 3], [4, 5]], np.int32)
    lens = np.array([3, 8, 6, 11], np.int32)
    counts = np.array([6, 6, 100, 6], np.int32)
    dk, dv = dev_array(kp), dev_array(vp)
    K.kv_append_paged(dev_array(k), dev_array(v), dk, dv, dev_array(table, "int32"), dev_array(lens, "int32"),
                      counts=dev_array(counts, "int32"))
    assert np.array_equal(host_pool(dk), ref.append(k, kp, table, lens, counts))
    assert np.array_equal(host_pool(dv), ref.append(v, vp, table, lens, counts))


# ---------------------------------------------------------------------------
# evict
# ---------------------------------------------------------------------------


def check_evict(lengths, keep, recent, Hkv=2, D=32, page=8, cache="float32", layout="heads", seed=0, weights=None,
                edit=None):
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(seed)
    B = len(lengths)
    cap_pages = max(1, max(-(-n // page) for n in lengths))
    width = -(-min(keep, cap_pages * page) // page)
    table, total, free = make_table(rng, lengths, page, spare=B * width + 1)
    to = free[:B * width].reshape(B, width).copy()
    kp, vp = (make_pool(rng, total, Hkv, page, D, cache) for _ in range(2))
    cap = table.shape[1] * page
    w = rng.random((B, Hkv, cap + 2), dtype=np.float32) if weights is None else weights(rng, (B, Hkv, cap + 2))
    a = dict(table=table, to=to, lengths=np.array(lengths, np.int32))
    if edit is not None:
        edit(a)
    dk, dv = (to_device(p, cache, layout) for p in (kp, vp))
    out = full(w.shape, 3.0)
    n, w_out, slots = K.kv_evict_paged(dk, dv, dev_array(a["table"], "int32"), dev_array(a["lengths"], "int32"),
                                       dev_array(w), dev_array(a["to"], "int32"), keep, recent, weights_out=out)
    e = ref.evict(kp, vp, a["table"], a["lengths"], w, a["to"], keep, recent)
    assert np.array_equal(host(slots), e[4])
    assert np.array_equal(host(n), e[2])
    assert np.array_equal(host(w_out)[..., :cap], e[3][..., :cap], equal_nan=True)
    assert np.all(host(w_out)[..., cap:] == 3.0)
    assert np.array_equal(host_pool(dk), e[0]) and np.array_equal(host_pool(dv), e[1])


@pytest.mark.parametrize("cache", ["float32", "bfloat16"])
@pytest.mark.parametrize("D,page,layout", [(16, 8, "rows"), (128, 16, "heads"), (64, 5, "rows")])
def test_evict_types_sizes_and_layouts(dev, cache, D, page, layout):
    check_evict([50, 17, 16, 3, 0, 255], 16, 4, D=D, page=page, cache=cache, layout=layout, seed=D)


@pytest.mark.parametrize("n,keep,recent", [(1, 1, 0), (1, 1, 1), (2, 1, 0), (2, 1, 1), (300, 299, 0), (300, 299, 299),
                                           (300, 1, 0), (300, 300, 10), (300, 500, 7), (2000, 777, 111),
                                           (5001, 1024, 64), (1025, 1024, 1024)])
def test_evict_sizes(dev, n, keep, recent):
    check_evict([n], keep, recent, Hkv=1, D=16, page=16, seed=n)


@pytest.mark.parametrize("kind", ["zeros", "few_values", "ascending", "descending", "signs", "specials", "tiny"])
def test_evict_weights(dev, kind):
    """Ties go to the lowest row; -0 equals 0, NaN counts above every number;
    subnormal weights differ from 0."""
    def weights(rng, shape):
        n = np.prod(shape)
        if kind == "zeros":
            return np.zeros(shape, np.float32)
        if kind == "few_values":
            return rng.integers(0, 3, shape).astype(np.float32)
        if kind in ("ascending", "descending"):
            w = np.arange(n, dtype=np.float32).reshape(shape)
            return w if kind == "ascending" else -w
        if kind == "signs":
            return rng.choice(np.array([-1.0, -0.0, 0.0, 1.0], np.float32), shape)
        if kind == "tiny":
            return rng.choice(np.array([0.0, 1e-45, 3e-45, 1e-39], np.float32), shape)
        return rng.choice(np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, 2.0], np.float32), shape)

    check_evict([400, 129, 64], 64, 16, seed=11, weights=weights)


def test_evict_long(dev):
    """More rows than one pass of a workgroup holds."""
    def weights(rng, shape):
        w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
        w[rng.random(shape) < 0.2] = 0
        return w

    check_evict([70001, 66000], 20000, 500, Hkv=1, D=16, page=64, cache="bfloat16", seed=12, weights=weights)


@pytest.mark.parametrize("n", [256, 257, 1024, 1025, 4096, 4097, 16384, 16385, 32768, 32769, 49152, 49153])
def test_evict_around_the_selections_sizes(dev, n):
    check_evict([n], n // 3, n // 50, Hkv=1, D=16, page=128, cache="bfloat16", seed=n)


@pytest.mark.parametrize("kind", ["sampled_large", "sampled_small", "two_halves", "one_value_but_few"])
@pytest.mark.parametrize("n,keep", [(20000, 5000), (20000, 300), (60000, 59000)])
def test_evict_where_a_sample_misleads(dev, kind, n, keep):
    """Rows that a selection samples say nothing, or the wrong thing, of the
    others; half the rows below the other half; nearly all of one weight."""
    def weights(rng, shape):
        w = rng.random(shape, dtype=np.float32)
        at = (np.arange(4096) * (n - 7)) // 4096
        if kind == "sampled_large":
            w[..., at] += 10
        elif kind == "sampled_small":
            w[..., at] -= 10
        elif kind == "two_halves":
            w[..., n // 2:] += 100
        else:
            w[:] = 0.5
            w[..., rng.integers(0, n, 50)] = 0.25
            w[..., rng.integers(0, n, 50)] = 0.75
        return w

    check_evict([n], keep, 7, Hkv=1, D=16, page=128, cache="bfloat16", seed=keep, weights=weights)


def test_evict_more_rows_between_than_are_listed(dev):
    check_evict([150000, 8000], 50000, 100, Hkv=1, D=16, page=64, cache="bfloat16", seed=15)


@pytest.mark.parametrize("B, Hkv, D, n, keep", [
    (6, 8, 128, 700, 500),   # 1536 workgroups: one launch
    (6, 8, 128, 700, 513),   # 1584: two
    (2, 8, 128, 2000, 512),  # 512
    (2, 8, 128, 2000, 520),  # 528
    (3, 8, 128, 250, 249),
])
def test_evict_many_heads(dev, B, Hkv, D, n, keep):
    check_evict([n - 13 * b for b in range(B)], keep, keep // 5, Hkv=Hkv, D=D, page=20, seed=n + keep)


def test_evict_pages_that_are_not_there(dev):
    """Kept rows of pages outside the pool become zeros; rows whose new page
    is outside it are dropped."""
    def edit(a):
        a["table"][0, 1] = -1
        a["table"][1, -1] = 10 ** 6
        a["to"][1, 0] = -1

    check_evict([40, 40], 24, 8, page=8, seed=13, edit=edit)


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------


def test_decoding_loop_with_eviction(dev):
    """Prompts appended, then steps that append a row, attend, accumulate the
    weights and cut the caches back when they pass the budget, between two page
    tables; every step against the plain forms on the same state."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(21)
    B, H, Hkv, D, page, keep, recent, room = 3, 4, 2, 64, 8, 24, 6, 32
    width = room // page
    ids = rng.permutation(2 * B * width).astype(np.int32)
    tables = [ids[:B * width].reshape(B, width), ids[B * width:].reshape(B, width)]
    dt = [dev_array(t, "int32") for t in tables]
    kp, vp = (make_pool(rng, 2 * B * width, Hkv, page, D, "bfloat16") for _ in range(2))
    dk, dv = dev_array(kp, "bfloat16"), dev_array(vp, "bfloat16")
    lens = np.array([20, 9, 24], np.int32)
    k, v = (rng.standard_normal((B, Hkv, 24, D), dtype=np.float32) for _ in range(2))
    K.kv_append_paged(dev_array(k), dev_array(v), dk, dv, dt[0], dev_array(lens, "int32"), counts=dev_array(lens, "int32"))
    kp, vp = (ref.append(bf16_round(x), p, tables[0], lens, lens) for x, p in ((k, kp), (v, vp)))
    dw = full((B, Hkv, room), 0.0)
    case = dict(q="float32", cache="bfloat16")
    at = 0
    for step in range(20):
        lens = lens + 1
        dl = dev_array(lens, "int32")
        q, k, v = (rng.standard_normal((B, h, 1, D), dtype=np.float32) for h in (H, Hkv, Hkv))
        K.kv_append_paged(dev_array(k), dev_array(v), dk, dv, dt[at], dl)
        kp, vp = (ref.append(bf16_round(x), p, tables[at], lens) for x, p in ((k, kp), (v, vp)))
        o, _ = K.attn_decode_paged(dev_array(q), dk, dv, dt[at], dl, 0.125, weights=dw, weights_in=dw)
        r = ref.decode(q, kp, vp, tables[at], lens, 0.125)
        assert np.all(np.abs(host(o) - r[0]) <= decode_bounds(case, r, room)[0]), step
        if lens.max() == room:
            w = host(dw)
            n, dw, slots = K.kv_evict_paged(dk, dv, dt[at], dl, dw, dt[1 - at], keep, recent)
            kp, vp, lens, w_out, want = ref.evict(kp, vp, tables[at], lens, w, tables[1 - at], keep, recent)
            assert np.array_equal(host(slots), want) and np.array_equal(host(n), lens)
            assert np.array_equal(host(dw), w_out)
            at = 1 - at
        assert np.array_equal(host_pool(dk), kp) and np.array_equal(host_pool(dv), vp), step


def test_recorded_step_follows_device_state(dev):
    """A recorded append and attention replay with lengths, table and rows that
    changed in device memory; two graphs recorded at different sizes run in
    turn, with eager calls between."""
    from minitorch_amd import kernels as K
    from minitorch_amd.graphs import Graph

    rng = np.random.default_rng(31)
    sets = []
    for B, H, Hkv, D, page, top in ((2, 4, 2, 64, 16, 3000), (3, 6, 6, 32, 10, 700)):
        table, total, _ = make_table(rng, [top] * B, page)
        kp, vp = (make_pool(rng, total, Hkv, page, D, "bfloat16") for _ in range(2))
        s = dict(table=table, kp=kp, vp=vp, dk=dev_array(kp, "bfloat16"), dv=dev_array(vp, "bfloat16"),
                 dt=dev_array(table, "int32"), dl=full((B,), 1, "int32"), w=full((B, Hkv, table.shape[1] * page), 0.0),
                 q=empty((B, H, 1, D)), k=empty((B, Hkv, 1, D)), v=empty((B, Hkv, 1, D)), lse=empty((B, H)),
                 out=empty((B, H, 1, D)), top=top)

        def call(s=s):
            K.kv_append_paged(s["k"], s["v"], s["dk"], s["dv"], s["dt"], s["dl"])
            K.attn_decode_paged(s["q"], s["dk"], s["dv"], s["dt"], s["dl"], 0.125, out=s["out"], lse=s["lse"],
                                weights=s["w"], weights_in=s["w"])

        s["call"], s["graph"] = call, Graph()
        sets.append(s)
    for s in sets:
        s["call"]()  # eager once, on rows the loop below writes again
        with s["graph"].capture():
            s["call"]()
        s["w"].fill_(0.0)
    for i in range(6):
        for s in sets:
            B = s["table"].shape[0]
            lens = rng.integers(1, s["top"] + 1, B).astype(np.int32)
            q, k, v = (rng.standard_normal(s[x].shape, dtype=np.float32) for x in "qkv")
            if i == 0:  # the eager call above appended row 0 from unset memory
                s["dk"].copy_(dev_array(s["kp"], "bfloat16"))
                s["dv"].copy_(dev_array(s["vp"], "bfloat16"))
            for name, x in (("q", q), ("k", k), ("v", v)):
                s[name].copy_(x)
            s["dl"].copy_(lens)
            before = host(s["w"])
            if i == 3:
                s["call"]()
            else:
                s["graph"].replay()
            s["kp"], s["vp"] = (ref.append(bf16_round(x), p, s["table"], lens) for x, p in ((k, s["kp"]), (v, s["vp"])))
            r = ref.decode(q, s["kp"], s["vp"], s["table"], lens, 0.125)
            ob, lb, rel = decode_bounds(dict(q="float32", cache="bfloat16"), r, s["top"])
            assert np.all(np.abs(host(s["out"]) - r[0]) <= ob), i
            assert np.all(np.abs(host(s["lse"]) - r[1]) <= lb), i
            got = host(s["w"]).astype(np.float64) - before
            G = rel.shape[1] // got.shape[1]
            relw = rel.reshape(B, -1, G).max(-1)[..., None]
            assert np.all(np.abs(got - r[2]) <= relw * r[2] + (G + 3) * U * (before + r[2])), i
            assert np.array_equal(host_pool(s["dk"]), s["kp"])


@pytest.mark.parametrize("q", ["float32", "bfloat16"])
@pytest.mark.parametrize("B,width", [(64, 1), (3, 300)])
def test_decode_weights_keep_fp32s_bits(dev, q, B, width):
    """Values that cancel show the weights' own precision behind bf16 outputs:
    three rows, the first of score 0 and value 0, the others' scores 2^-12 apart
    and their values each other's negatives, so that o is some 2^-12 of sum p|v|.
    The scores are exact in fp32.  A weight is then off by 3 u |s| (the scale's
    two roundings and the product's; |s| <= 1.5), 2 u (the exponential) and u (its
    pieces), the sums and the quotient by 8 u: below 16 u, or 2^-20, of sum p|v|
    in all, and a bf16 output by half a step 2^-8 of itself besides.  Two bf16
    pieces of a weight would be off by up to 2^-16 of it."""
    from minitorch_amd import kernels as K

    rng = np.random.default_rng(B)
    H, D, page = 16, 16, 16
    a = bf16_round(rng.uniform(0.5, 1, (B, H)).astype(np.float32))
    b = bf16_round(rng.uniform(0.25, 1.5, B).astype(np.float32))
    v = bf16_round(rng.uniform(1, 2, (B, D)).astype(np.float32))
    qs = np.zeros((B, H, 1, D), np.float32)
    qs[:, :, 0, 0], qs[:, :, 0, 1] = a, 2.0 ** -6
    kp, vp = (np.zeros((B, 1, page, D), np.float32) for _ in range(2))
    kp[:, 0, 1:3, 0] = -b[:, None]
    kp[:, 0, 2, 1] = -2.0 ** -6
    vp[:, 0, 1], vp[:, 0, 2] = v, -v
    table = np.full((B, width), -1, np.int32)
    table[:, 0] = rng.permutation(B)
    kp[table[:, 0]], vp[table[:, 0]] = kp.copy(), vp.copy()
    lens = np.full(B, 3, np.int32)
    o, _ = K.attn_decode_paged(dev_array(qs, q), dev_array(kp, "bfloat16"), dev_array(vp, "bfloat16"),
                               dev_array(table, "int32"), dev_array(lens, "int32"), 1.0)
    want, _, _, _, pv = ref.decode(qs, kp, vp, table[:, :1], lens, 1.0)
    assert np.abs(want).max() < 2.0 ** -10 * pv.max()
    bound = 2.0 ** -20 * pv + (2.0 ** -8 if q == "bfloat16" else 0) * np.abs(want)
    off = np.abs(host(o) - want) / bound
    assert off.max() <= 1, float(off.max())


def test_evict_weights_wider_than_the_table(dev):
    """Columns behind the table's rows: 0 where the call makes the new weights
    itself, left as they were in a caller's; a wider table then counts from there."""
    from minitorch_amd import device, kernels as K

    rng = np.random.default_rng(17)
    B, Hkv, D, page, keep = 2, 2, 16, 4, 6
    kp, vp = (make_pool(rng, 12, Hkv, page, D, "float32") for _ in range(2))
    dk, dv = dev_array(kp), dev_array(vp)
    table, to = np.array([[0, 1], [2, 3]], np.int32), np.array([[4, 5, 6, -1], [7, 8, 9, -1]], np.int32)
    lens = np.array([8, 5], np.int32)
    w = rng.random((B, Hkv, 16), dtype=np.float32)
    args = (dk, dv, dev_array(table, "int32"), dev_array(lens, "int32"), dev_array(w), dev_array(to, "int32"), keep, 2)
    device.empty_cache()
    junk = [full(w.shape, 7.0) for _ in range(4)]  # what freed memory holds
    del junk
    n, w_out, _ = K.kv_evict_paged(*args)
    got = host(w_out)
    assert not got[..., 8:].any()
    n = host(n)
    assert n.tolist() == [6, 5]
    assert np.all(host(K.kv_evict_paged(*args, weights_out=full(w.shape, 3.0))[1])[..., 8:] == 3.0)
    # two rows more each, in the wider table
    lens = (n + 5).astype(np.int32)
    q = rng.standard_normal((B, Hkv, 1, D), dtype=np.float32)
    K.attn_decode_paged(dev_array(q), dk, dv, dev_array(to, "int32"), dev_array(lens, "int32"), 0.2, weights=w_out,
                        weights_in=w_out)
    r = ref.decode(q, host_pool(dk), host_pool(dv), to, lens, 0.2)
    assert np.abs(host(w_out) - got - r[2]).max() <= 1e-5


def test_calls_on_another_stream(dev):
    """Append, attention, eviction and log probabilities launched on a stream
    of their own: the null stream's bits."""
    import ctypes

    from minitorch_amd import _lib as L, device, kernels as K

    rng = np.random.default_rng(51)
    B, H, Hkv, D, page = 3, 4, 2, 64, 16
    lens = [3000, 17, 700]
    table, total, free = make_table(rng, lens, page, spare=3 * 16)
    kp, vp = (make_pool(rng, total, Hkv, page, D, "bfloat16") for _ in range(2))
    new = rng.standard_normal((2, B, Hkv, 1, D), dtype=np.float32)
    q = dev_array(rng.standard_normal((B, H, 1, D), dtype=np.float32))
    dk, dv = dev_array(new[0]), dev_array(new[1])
    dt, dl = dev_array(table, "int32"), dev_array(np.array(lens, np.int32), "int32")
    to = dev_array(free[:48].reshape(3, 16).copy(), "int32")
    x = dev_array(rng.standard_normal((9, 5000), dtype=np.float32))
    tok, g = dev_array(rng.integers(0, 5000, 9), "int64"), dev_array(rng.standard_normal(9).astype(np.float32))

    def work():
        a, b = dev_array(kp, "bfloat16"), dev_array(vp, "bfloat16")
        w = full((B, Hkv, table.shape[1] * page), 0.0)
        K.kv_append_paged(dk, dv, a, b, dt, dl)
        lse = empty((B, H))
        o, _ = K.attn_decode_paged(q, a, b, dt, dl, 0.125, lse=lse, weights=w)
        out = [a, b, o, lse, w, *K.kv_evict_paged(a, b, dt, dl, w, to, 256, 32)]
        lp = K.token_logprobs(x, tok, top=7)
        return out + [*lp, K.token_logprobs_bwd(x, tok, lp[2], lp[1], g, g)]

    want = [host(t) for t in work()]
    device.synchronize()
    stream = ctypes.c_void_p()
    L.call("mtx_stream_create", ctypes.byref(stream))
    try:
        L._STREAM[0] = stream
        out = work()
        L.call("mtx_stream_sync", stream)
    finally:
        L._STREAM[0] = None
        L.call("mtx_stream_destroy", stream)
    for a, b in zip(out, want):
        assert np.array_equal(host(a), b, equal_nan=True)
