"""What the operators of training with a large vocabulary take and refuse at the ends
of their ranges.  No GPU: every check runs before any HIP call."""
import pytest
from test_vocab_refusals import Fake, _kernels, call, dropout, p, xent

from minitorch_amd import _lib as L


@pytest.mark.parametrize("over,code,frag", [
    (dict(rows=1, cols=(1 << 32) + 8), L.MTX_ERR_ARG, "overlap"),  # rows of 8 values in between
    (dict(rows=1, cols=(1 << 33) + 8, ldx=1 << 34, ldy=1 << 34), L.MTX_ERR_SHAPE, "2^33"),
    (dict(rows=3, cols=(1 << 32) - 8, ldx=1 << 32, ldy=1 << 32), L.MTX_ERR_SHAPE, "2^33"),
    # up to there the next check is reached
    (dict(rows=1, cols=1 << 33, ldx=1 << 33, ldy=1 << 33, x=None), L.MTX_ERR_ARG, "null"),
    (dict(rows=1, cols=1 << 31, ldx=1 << 31, ldy=1 << 31, base=p(12)), L.MTX_ERR_ARG, "aligned"),
])
def test_dropout_of_rows_longer_than_32_bits(over, code, frag):
    rc, msg = dropout(over)
    assert rc == code and frag in msg, (rc, msg)


def test_dropout_wrapper_passes_all_columns(monkeypatch):
    K = _kernels(monkeypatch)
    seen = []
    monkeypatch.setattr(Fake, "data_ptr", lambda self: 16)
    monkeypatch.setattr(L, "call", lambda name, *args: seen.append((name, args)))
    n = (1 << 32) + 8
    K.dropout(Fake((1, n)), 0.5, 1, out=Fake((1, n)))
    name, args = seen[0]
    types = L.SIGNATURES[name][1]
    assert name == "mtx_dropout" and [t(a).value for t, a in zip(types, args)][7:9] == [1, n]


FAR = (1 << 32) + 8  # wrapped to 32 bits: 8


@pytest.mark.parametrize("call,frag", [
    (lambda K: K.embedding_lookup(Fake((3, FAR)), Fake((4,), "int64"), out=Fake((4, FAR))), "C must"),
    (lambda K: K.embedding_grad(Fake((4,), "int64"), Fake((4, FAR)), Fake((3, FAR))), "C must"),
    (lambda K: K.linear_xent(Fake((4, FAR)), Fake((FAR, 10)), Fake((4,), "int64")), "C must"),
    (lambda K: K.linear_xent(Fake((4, 8)), Fake((8, FAR)), Fake((4,), "int64")), "V must"),
    (lambda K: K.linear_xent(Fake((4, 8)), Fake((8, 1 << 31)), Fake((4,), "int64")), "V must"),
])
def test_sizes_that_the_library_takes_as_32_bits(monkeypatch, call, frag):
    K = _kernels(monkeypatch)
    monkeypatch.setattr(L, "call", lambda *args: pytest.fail("wrapped and passed on"))
    monkeypatch.setattr(Fake, "data_ptr", lambda self: 16)
    with pytest.raises(ValueError, match=frag):
        call(K)


@pytest.mark.parametrize("over", [dict(gdt=256), dict(dtype=0, gdt=257), dict(gdt=258), dict(gdt=513)])
def test_one_piece_is_for_bf16_gradients(over):
    rc, msg = xent(over)
    assert rc == L.MTX_ERR_DTYPE and "gradients" in msg


def test_one_piece_wrapper_refuses(monkeypatch):
    K = _kernels(monkeypatch)
    args = Fake((4, 8), "bfloat16"), Fake((8, 10), "bfloat16"), Fake((4,), "int64")
    for grads in ({}, dict(dx=Fake((4, 8))), dict(bias=Fake((10,)), db=Fake((10,)))):
        with pytest.raises(ValueError, match="one_piece"):
            K.linear_xent(*args, one_piece=True, **grads)


def test_one_piece_takes_less_workspace():
    f = L.lib().mtx_linear_xent_workspace_bytes
    one, two, three = (f(1, g, 4096, 64, 1000, 1, 1 << 30) for g in (257, 1, 0))
    # 4096 x 1024 values of two bytes a piece
    assert two - one >= 1 << 23 and three - two >= 1 << 23


@pytest.mark.parametrize("V,C", [(10, 384), (65, 384), (128, 256), (255, 128), (255, 256), (128, 1024), (255, 4096)])
def test_small_tables_workspace_does_not_grow_with_the_tokens(V, C):
    """The chunks' tables of as many workgroups as the chip's LDS holds (256 x 160 KB) and
    one more chunk's, or the sorted way's pieces and lists: a quarter of the gradient's
    rows in fp32, twelve bytes a token and eight a table row."""
    f = L.lib().mtx_embedding_grad_workspace_bytes
    for n in (1 << 15, 1 << 17, 1 << 20, 1 << 22):
        for dtype in (0, 1):
            most = max(256 * 163840 + V * C * 4, (n // 32 + 1) * 8 * C + 12 * n + 8 * V + 2048)
            assert f(dtype, n, V, C) <= most, (n, dtype)
    assert f(0, 1 << 22, V, C) == f(1, 1 << 22, V, C)


@pytest.mark.parametrize("n,C,V", [(12000, 64, 100), (6000, 100, 120), (9000, 40, 500), (3001, 64, 97)])
def test_fp32_weights_gradients_have_room_for_all_ranges_of_the_rows(n, C, V):
    """The product dW = x^T dz asks for this many ranges of the rows (the fp32 tiles' rule),
    each with its C + 1 rows of V sums, and is not cut at all without the room."""
    tiles = -(-C // 64) * -(-V // 64)
    ranges = min(64 if n >= 4096 else 16, -(-768 // tiles), n // 256)
    kept = n * (-(-V // 32) * 32) * 4  # the logits
    f = L.lib().mtx_linear_xent_workspace_bytes
    assert f(0, 0, n, C, V, 0, 1 << 30) >= kept + ranges * (C + 1) * V * 4


@pytest.mark.parametrize("over,code,frag", [
    (dict(rows=-1), L.MTX_ERR_ARG, "rows"), (dict(cols=0), L.MTX_ERR_ARG, "cols"), (dict(ld=7), L.MTX_ERR_ARG, "ld"),
    (dict(p=1.0), L.MTX_ERR_ARG, "p="), (dict(keep=None), L.MTX_ERR_ARG, "null"), (dict(base=p(12)), L.MTX_ERR_ARG, "aligned"),
    (dict(rows=1 << 60), L.MTX_ERR_SHAPE, "large"),
])
def test_dropout_keep_refusals(over, code, frag):
    rc, msg = call("mtx_dropout_keep", dict(keep=p(16), rows=4, cols=8, ld=8, p=0.5, seed=1, offset=0, sub=0, base=None,
                                            stream=None), over)
    assert rc == code and frag in msg, (rc, msg)


@pytest.mark.parametrize("n", [8192, 100000])
@pytest.mark.parametrize("grads,pieces", [(257, 1), (1, 2), (0, 3)])
def test_workspace_is_what_the_documents_say(n, grads, pieces):
    """The logits, half as much again for a piece of their gradient, copies of x and w, a
    sum of dw where there are several blocks, and the sums of ranges of the last tiles, for
    these sizes fewer than four tiles of 256 x 128 for each of the 512 places."""
    C, V = 1024, 50021
    f = L.lib().mtx_linear_xent_workspace_bytes
    for logits in (1 << 28, 1 << 31):
        rows = min(n, logits // (4 * 50048) // 256 * 256)
        kept = rows * 50048 * 4
        got = f(1, grads, n, C, V, 0, logits)
        copies = 2 * (rows + 50048) * C + (4 * C * V if rows < n and grads != 0 else 0)
        assert kept * (1 + pieces / 2) <= got <= kept * (1 + pieces / 2) + copies + 4 * 512 * 256 * 128 * 4, (got, kept)


@pytest.mark.parametrize("base,frag", [(Fake((1,), "int32"), "base"), (Fake((2,), "int64"), "base")])
def test_keep_mask_wrapper_refuses(monkeypatch, base, frag):
    K = _kernels(monkeypatch)
    monkeypatch.setattr(Fake, "fill_", lambda self, value: self, raising=False)
    with pytest.raises(ValueError, match=frag):
        K.dropout_keep_philox((1, 2, 3, 4), 0.5, 1, 0, base=base)
