"""What the operators of training with a large vocabulary refuse: every check runs
on the host before any HIP call, so fake addresses do.  And their float64 forms
against differences."""
import ctypes as C

import numpy as np
import pytest

from minitorch_amd import _lib as L
from oracle import vocab as ref

BIG = 1 << 40


def p(x):
    return C.c_void_p(x) if x else None


def call(fn, args, over):
    assert set(over) <= set(args), over
    rc = getattr(L.lib(), fn)(*{**args, **over}.values())
    return rc, L.lib().mtx_last_error().decode()


def lookup(over):
    return call("mtx_embedding_lookup", dict(dtype=0, out_dtype=0, w=p(16), ldw=8, V=10, ids=p(16), n=4, C=8, scale=1.0,
                                             out=p(16), ldo=8, stream=None), over)


def grad(over):
    return call("mtx_embedding_grad", dict(dtype=0, ids=p(16), n=4, g=p(16), ldg=8, scale=1.0, dw=p(16), lddw=8, V=10,
                                           C=8, acc=0, ws=p(256), ws_bytes=BIG, stream=None), over)


def dropout(over):
    return call("mtx_dropout", dict(dtype=0, x=p(16), ldx=8, res=None, ldr=0, y=p(16), ldy=8, rows=4, cols=8, p=0.5,
                                    scale=2.0, seed=1, offset=0, sub=0, base=None, stream=None), over)


def xent(over):
    return call("mtx_linear_xent", dict(
        dtype=1, gdt=1, n=4, C=8, V=10, x=p(16), ldx=8, w=p(16), swc=10, swv=1, bias=p(16), labels=p(16), loss=p(16),
        row=p(16), lse=p(16), dx=p(16), lddx=8, dw=p(16), sdc=10, sdv=1, db=p(16), logits=1 << 20, ws=p(256),
        ws_bytes=BIG, stream=None), over)


@pytest.mark.parametrize("fn,over,code,frag", [
    (lookup, dict(dtype=2), L.MTX_ERR_DTYPE, "dtype"),
    (lookup, dict(out_dtype=-1), L.MTX_ERR_DTYPE, "dtype"),
    (lookup, dict(n=-1), L.MTX_ERR_SHAPE, "n"),
    (lookup, dict(n=1 << 31), L.MTX_ERR_SHAPE, "2^31"),
    (lookup, dict(V=0), L.MTX_ERR_SHAPE, "V"),
    (lookup, dict(C=0), L.MTX_ERR_SHAPE, "C"),
    (lookup, dict(ldw=7), L.MTX_ERR_ARG, "overlap"),
    (lookup, dict(ldo=7), L.MTX_ERR_ARG, "overlap"),
    (lookup, dict(w=None), L.MTX_ERR_ARG, "null"),
    (lookup, dict(ids=None), L.MTX_ERR_ARG, "null"),
    (lookup, dict(out=None), L.MTX_ERR_ARG, "null"),
    (grad, dict(dtype=2), L.MTX_ERR_DTYPE, "dtype"),
    (grad, dict(n=-1), L.MTX_ERR_SHAPE, "n"),
    (grad, dict(V=(1 << 31) - 1023), L.MTX_ERR_SHAPE, "1024"),
    (grad, dict(n=1 << 31), L.MTX_ERR_SHAPE, "2^31"),
    (grad, dict(V=0), L.MTX_ERR_SHAPE, "V"),
    (grad, dict(C=0), L.MTX_ERR_SHAPE, "C"),
    (grad, dict(ldg=7), L.MTX_ERR_ARG, "overlap"),
    (grad, dict(lddw=7), L.MTX_ERR_ARG, "overlap"),
    (grad, dict(ids=None), L.MTX_ERR_ARG, "null"),
    (grad, dict(g=None), L.MTX_ERR_ARG, "null"),
    (grad, dict(dw=None), L.MTX_ERR_ARG, "null"),
    (dropout, dict(dtype=3), L.MTX_ERR_DTYPE, "dtype"),
    (dropout, dict(rows=-1), L.MTX_ERR_SHAPE, "rows"),
    (dropout, dict(cols=0), L.MTX_ERR_SHAPE, "cols"),
    (dropout, dict(p=1.0), L.MTX_ERR_ARG, "p="),
    (dropout, dict(p=-0.1), L.MTX_ERR_ARG, "p="),
    (dropout, dict(p=float("nan")), L.MTX_ERR_ARG, "p="),
    (dropout, dict(ldx=7), L.MTX_ERR_ARG, "overlap"),
    (dropout, dict(ldy=7), L.MTX_ERR_ARG, "overlap"),
    (dropout, dict(res=p(16), ldr=7), L.MTX_ERR_ARG, "overlap"),
    (dropout, dict(x=None), L.MTX_ERR_ARG, "null"),
    (dropout, dict(y=None), L.MTX_ERR_ARG, "null"),
    (dropout, dict(base=p(12)), L.MTX_ERR_ARG, "aligned"),
    (dropout, dict(rows=1 << 31, cols=8), L.MTX_ERR_SHAPE, "2^33"),
    (xent, dict(dtype=4), L.MTX_ERR_DTYPE, "dtype"),
    (xent, dict(gdt=2), L.MTX_ERR_DTYPE, "gradients"),
    (xent, dict(dtype=0), L.MTX_ERR_DTYPE, "gradients"),
    (xent, dict(n=-1), L.MTX_ERR_SHAPE, "n"),
    (xent, dict(C=0), L.MTX_ERR_SHAPE, "C"),
    (xent, dict(C=(1 << 20) + 1, ldx=1 << 21), L.MTX_ERR_SHAPE, "C"),
    (xent, dict(V=0), L.MTX_ERR_SHAPE, "V"),
    (xent, dict(V=(1 << 27) + 1), L.MTX_ERR_SHAPE, "V"),
    (xent, dict(ldx=7), L.MTX_ERR_ARG, "overlap"),
    (xent, dict(swc=9), L.MTX_ERR_ARG, "stride"),
    (xent, dict(swc=2, swv=10), L.MTX_ERR_ARG, "stride"),
    (xent, dict(swc=1, swv=7), L.MTX_ERR_ARG, "stride"),
    (xent, dict(sdc=9), L.MTX_ERR_ARG, "stride"),
    (xent, dict(sdc=1, sdv=7), L.MTX_ERR_ARG, "stride"),
    (xent, dict(lddx=7), L.MTX_ERR_ARG, "overlap"),
    (xent, dict(bias=None), L.MTX_ERR_ARG, "bias"),
    (xent, dict(x=None), L.MTX_ERR_ARG, "null"),
    (xent, dict(w=None), L.MTX_ERR_ARG, "null"),
    (xent, dict(labels=None), L.MTX_ERR_ARG, "null"),
    (xent, dict(loss=None), L.MTX_ERR_ARG, "null"),
    (xent, dict(row=None), L.MTX_ERR_ARG, "null"),
    (xent, dict(lse=None), L.MTX_ERR_ARG, "null"),
    (xent, dict(V=1 << 22, swc=1 << 22, sdc=1 << 22), L.MTX_ERR_ARG, "2^22"),
    (xent, dict(lddx=1 << 26), L.MTX_ERR_ARG, "2^26"),
    (xent, dict(sdc=1 << 26), L.MTX_ERR_ARG, "2^26"),
    (xent, dict(logits=0), L.MTX_ERR_ARG, "logits_bytes"),
    (xent, dict(ws=None), L.MTX_ERR_ARG, "workspace"),
    (xent, dict(ws=p(128)), L.MTX_ERR_ARG, "workspace"),
    (xent, dict(ws_bytes=300), L.MTX_ERR_ARG, "workspace"),
])
def test_refusals(fn, over, code, frag):
    rc, msg = fn(over)
    assert rc == code and frag in msg, (rc, msg)


class Fake:
    """A device array of given shape, strides and dtype at no address."""
    is_cuda = True

    def __init__(self, shape, dtype="float32", strides=None):
        self.shape, self.dtype = tuple(shape), dtype
        acc, st = 1, []
        for s in self.shape[::-1]:
            st.append(acc)
            acc *= s
        self._strides = tuple(st[::-1]) if strides is None else strides

    def stride(self, d=None):
        return self._strides if d is None else self._strides[d]

    def data_ptr(self):
        raise AssertionError("checked before any address is taken")

    def numel(self):
        return int(np.prod(self.shape))


def _kernels(monkeypatch):
    from minitorch_amd import device, kernels

    monkeypatch.setattr(device, "device", lambda: 0)
    monkeypatch.setattr(device, "empty_buf", lambda shape, dtype="float32": Fake(shape, dtype))
    return kernels


@pytest.mark.parametrize("over,frag", [
    (dict(ids=Fake((4,), "int32")), "ids"),
    (dict(ids=Fake((2, 2), "int64")), "ids"),
    (dict(ids=Fake((4,), "int64", (2,))), "ids"),
    (dict(weight=Fake((10, 8), "float32", (8, 2))), "rows"),
    (dict(weight=Fake((10, 8), "float32", (4, 1))), "overlap"),
    (dict(weight=Fake((10, 8), "int32")), "dtype"),
    (dict(out=Fake((4, 9))), "out"),
    (dict(out=Fake((5, 8))), "out"),
    (dict(out=Fake((4, 8), "int64")), "dtype"),
])
def test_lookup_wrapper_refuses(monkeypatch, over, frag):
    K = _kernels(monkeypatch)
    with pytest.raises(ValueError, match=frag):
        K.embedding_lookup(**{**dict(weight=Fake((10, 8)), ids=Fake((4,), "int64"), out=Fake((4, 8))), **over})


@pytest.mark.parametrize("over,frag", [
    (dict(ids=Fake((4,), "int32")), "ids"),
    (dict(grad=Fake((5, 8))), "grad"),
    (dict(grad=Fake((4, 8), "uint8")), "dtype"),
    (dict(dweight=Fake((10, 8), "bfloat16")), "fp32"),
    (dict(dweight=Fake((10, 8), "float32", (1, 10))), "rows"),
    (dict(dweight=Fake((0, 8))), "no rows"),
])
def test_grad_wrapper_refuses(monkeypatch, over, frag):
    K = _kernels(monkeypatch)
    with pytest.raises(ValueError, match=frag):
        K.embedding_grad(**{**dict(ids=Fake((4,), "int64"), grad=Fake((4, 8)), dweight=Fake((10, 8))), **over})


@pytest.mark.parametrize("over,frag", [
    (dict(p=1.0), "probability"),
    (dict(p=float("nan")), "probability"),
    (dict(x=Fake((4, 8, 2))), "rows, cols"),
    (dict(x=Fake((4, 8), "int32")), "dtype"),
    (dict(residual=Fake((4, 9))), "residual"),
    (dict(residual=Fake((4, 8), "bfloat16")), "residual"),
    (dict(out=Fake((4, 8), "bfloat16")), "out"),
    (dict(base=Fake((1,), "int32")), "base"),
    (dict(base=Fake((2,), "int64")), "base"),
])
def test_dropout_wrapper_refuses(monkeypatch, over, frag):
    K = _kernels(monkeypatch)
    with pytest.raises(ValueError, match=frag):
        K.dropout(**{**dict(x=Fake((4, 8)), p=0.5, seed=1), **over})


@pytest.mark.parametrize("over,frag", [
    (dict(w=Fake((9, 10))), "w must"),
    (dict(w=Fake((8, 10), "bfloat16")), "w must"),
    (dict(w=Fake((8, 10), "float32", (20, 2))), "contiguous"),
    (dict(x=Fake((4, 8), "float32", (1, 4))), "rows"),
    (dict(labels=Fake((5,), "int64")), "labels"),
    (dict(labels=Fake((4,), "int32")), "labels"),
    (dict(bias=Fake((9,))), "bias"),
    (dict(bias=Fake((10,), "bfloat16")), "bias"),
    (dict(db=Fake((10,))), "without a bias"),
    (dict(dx=Fake((4, 9))), "dx"),
    (dict(dx=Fake((4, 8), "bfloat16")), "gradients"),
    (dict(dw=Fake((8, 10), "float32", (30, 2))), "contiguous"),
    (dict(dx=Fake((4, 8)), dw=Fake((8, 10), "bfloat16")), "share"),
    (dict(loss=Fake((2,))), "loss"),
    (dict(logits_bytes=0), "logits_bytes"),
])
def test_xent_wrapper_refuses(monkeypatch, over, frag):
    K = _kernels(monkeypatch)
    with pytest.raises(ValueError, match=frag):
        K.linear_xent(**{**dict(x=Fake((4, 8)), w=Fake((8, 10)), labels=Fake((4,), "int64")), **over})


@pytest.mark.parametrize("fn,over,frag", [
    (lookup, dict(), "out is the table"),
    (grad, dict(), "dweight is grad"),
    (xent, dict(), "an output is an input"),
    (xent, dict(x=p(32), w=p(48), bias=p(64), dw=p(48)), "an output is an input"),
    (xent, dict(x=p(32), w=p(48), bias=p(64), loss=p(64)), "an output is an input"),
])
def test_outputs_in_place_of_inputs(fn, over, frag):
    rc, msg = fn(over)
    assert rc == L.MTX_ERR_ARG and frag in msg


def test_wrappers_refuse_host_arrays(monkeypatch):
    K = _kernels(monkeypatch)
    host = Fake((4, 8))
    host.is_cuda = False
    vec = Fake((10,))
    vec.is_cuda = False
    wide = Fake((8, 10))
    wide.is_cuda = False
    args = Fake((4, 8)), Fake((8, 10)), Fake((4,), "int64")
    for f in (lambda: K.dropout(Fake((4, 8)), 0.5, 1, residual=host), lambda: K.dropout(Fake((4, 8)), 0.5, 1, out=host),
              lambda: K.linear_xent(*args, bias=vec), lambda: K.linear_xent(*args, dx=host),
              lambda: K.linear_xent(*args, dw=wide), lambda: K.linear_xent(*args, bias=Fake((10,)), db=vec),
              lambda: K.embedding_grad(Fake((4,), "int64"), Fake((4, 8)), wide),
              lambda: K.dropout(host, 0.5, 1), lambda: K.embedding_lookup(host, Fake((4,), "int64")),
              lambda: K.embedding_grad(Fake((4,), "int64"), host, Fake((10, 8))),
              lambda: K.linear_xent(host, Fake((8, 10)), Fake((4,), "int64"))):
        with pytest.raises(ValueError, match="device arrays"):
            f()


def test_workspace_grows_with_the_rows_kept():
    f = L.lib().mtx_linear_xent_workspace_bytes
    few, many = (f(1, 1, 4096, 64, 1000, 1, b) for b in (1 << 20, 1 << 30))
    assert 0 < few < many < f(1, 0, 4096, 64, 1000, 1, 1 << 30)
    assert f(1, 1, -1, 64, 1000, 1, 1 << 20) == 0


# ---------------------------------------------------------------------------
# the oracle's own forms
# ---------------------------------------------------------------------------

def test_oracle_gradients_against_differences():
    rng = np.random.default_rng(0)
    x, w, b = rng.standard_normal((6, 5)), rng.standard_normal((5, 9)), rng.standard_normal(9)
    labels = np.array([0, 8, -1, 3, 3, 12])
    r = ref.linear_xent(x, w, labels, b)
    for arg, g in ((0, r["dx"]), (1, r["dw"]), (2, r["db"])):
        d = rng.standard_normal(g.shape)
        vals = []
        for s in (1e-6, -1e-6):
            a = [x.copy(), w.copy(), b.copy()]
            a[arg] += s * d
            vals.append(ref.linear_xent(a[0], a[1], labels, a[2])["loss"])
        assert abs((vals[0] - vals[1]) / 2e-6 - (g * d).sum()) < 1e-8


def test_oracle_lookup_gradient_is_the_transpose():
    rng = np.random.default_rng(1)
    w, ids, g = rng.standard_normal((7, 3)), rng.integers(-1, 8, 30), rng.standard_normal((30, 3))
    assert abs((ref.lookup(w, ids, 2.0) * g).sum() - (w * ref.lookup_grad(ids, g, 7, 2.0)[0]).sum()) < 1e-12


def test_oracle_keep_is_the_attention_masks():
    from oracle import philox

    for args in ((0.3, 12345678901, 7), (0.0, 1, (1 << 32) - 3)):
        assert np.array_equal(ref.keep((11, 13), *args), philox.keep_mask(11, 13, *args).astype(bool))
    assert not np.array_equal(ref.keep((11, 13), 0.5, 1), ref.keep((11, 13), 0.5, 1, 0, 1))
