"""What the paged cache's operators and the token log probabilities refuse:
every check runs on the host before any HIP call, so fake addresses do."""
import ctypes as C

import pytest

from minitorch_amd import _lib as L

I64x4 = C.c_int64 * 4
BIG = 1 << 40


def p(x):
    return C.c_void_p(x) if x else None


def call(fn, args, over):
    assert set(over) <= set(args), over
    args = {**args, **over}
    conv = [I64x4(*v) if isinstance(v, tuple) else v for v in args.values()]
    rc = getattr(L.lib(), fn)(*conv)
    return rc, L.lib().mtx_last_error().decode()


POOL = dict(n_pages=10, page=8, kp=p(256), kps=(2048, 512, 64, 1), vp=p(512), vps=(2048, 512, 64, 1))


def append(over):
    return call("mtx_kv_append_paged", dict(
        dtype=0, cache=0, B=2, T=3, H=4, D=64, k=p(16), ks=(768, 64, 256, 1), v=p(32), vs=(768, 64, 256, 1), **POOL,
        table=p(64), ld=5, width=5, lengths=p(128), counts=None, stream=None), over)


def decode(over):
    return call("mtx_attn_decode_paged", dict(
        dtype=0, cache=0, B=2, H=8, Hkv=4, D=64, q=p(16), qs=(512, 64, 0, 1), **POOL, table=p(64), ld=5, width=5,
        lengths=p(128), o=p(16), os=(512, 64, 0, 1), lse=None, win=None, w=None, wld=0, ws=p(1024), ws_bytes=BIG,
        scale=0.125, stream=None), over)


def evict(over):
    return call("mtx_kv_evict_paged", dict(
        cache=0, B=2, H=4, D=64, **POOL, table=p(64), ld=5, width=5, lengths=p(128), w=p(256), wld=40, to=p(2048),
        to_ld=2, to_pages=2, keep=16, recent=4, lengths_out=p(512), w_out=p(1024), slots=p(4096), stream=None), over)


CACHE = [
    (dict(D=48), L.MTX_ERR_SHAPE, "head dim"),
    (dict(B=0), L.MTX_ERR_SHAPE, ">= 1"),
    (dict(page=0), L.MTX_ERR_SHAPE, "pages"),
    (dict(page=65537), L.MTX_ERR_SHAPE, "pages"),
    (dict(n_pages=0), L.MTX_ERR_SHAPE, "pages"),
    (dict(n_pages=1 << 31), L.MTX_ERR_SHAPE, "pages"),
    (dict(width=0), L.MTX_ERR_SHAPE, "rows"),
    (dict(width=1 << 26), L.MTX_ERR_SHAPE, "rows"),
    (dict(table=None), L.MTX_ERR_ARG, "table"),
    (dict(lengths=None), L.MTX_ERR_ARG, "lengths"),
    (dict(ld=-1), L.MTX_ERR_ARG, "table"),
    (dict(kp=None), L.MTX_ERR_ARG, "null"),
    (dict(vp=p(520)), L.MTX_ERR_ARG, "aligned"),
    (dict(kps=(2048, 512, 64, 2)), L.MTX_ERR_ARG, "d stride"),
    (dict(vps=(2048, 512, 66, 1)), L.MTX_ERR_ARG, "multiple"),
    (dict(vps=(2048, -512, 64, 1)), L.MTX_ERR_ARG, "multiple"),
]


@pytest.mark.parametrize("fn", [append, decode, evict])
@pytest.mark.parametrize("over,code,frag", CACHE)
def test_cache_checks(fn, over, code, frag):
    rc, msg = fn(over)
    assert (rc, frag in msg) == (code, True), msg


@pytest.mark.parametrize("fn", [append, evict])
@pytest.mark.parametrize("strides", [(2048, 512, 0, 1), (1024, 512, 64, 1), (2048, 32, 64, 1), (0, 512, 64, 1)])
def test_pools_that_are_written_must_not_overlap(fn, strides):
    rc, msg = fn(dict(kps=strides))
    assert rc == L.MTX_ERR_ARG and "overlap" in msg


@pytest.mark.parametrize("over,code,frag", [
    (dict(dtype=1), L.MTX_ERR_DTYPE, "cache"),
    (dict(cache=7), L.MTX_ERR_DTYPE, "cache"),
    (dict(T=0), L.MTX_ERR_SHAPE, "at least 1"),
    (dict(T=1 << 30), L.MTX_ERR_SHAPE, "rows"),
    (dict(k=None), L.MTX_ERR_ARG, "null"),
    (dict(vs=(768, 64, 255, 1)), L.MTX_ERR_ARG, "multiple"),
])
def test_append_checks(over, code, frag):
    rc, msg = append(over)
    assert (rc, frag in msg) == (code, True), msg


@pytest.mark.parametrize("over,code,frag", [
    (dict(dtype=1), L.MTX_ERR_DTYPE, "cache"),
    (dict(H=6), L.MTX_ERR_SHAPE, "multiple"),
    (dict(Hkv=0), L.MTX_ERR_SHAPE, "multiple"),
    (dict(q=p(20)), L.MTX_ERR_ARG, "aligned"),
    (dict(os=(512, 32, 0, 1)), L.MTX_ERR_ARG, "overlap"),
    (dict(os=(0, 64, 0, 1)), L.MTX_ERR_ARG, "overlap"),
    (dict(scale=0.0), L.MTX_ERR_ARG, "scale"),
    (dict(scale=float("nan")), L.MTX_ERR_ARG, "scale"),
    (dict(win=p(64)), L.MTX_ERR_ARG, "weights_in"),
    (dict(w=p(64), wld=39), L.MTX_ERR_ARG, "40"),
    (dict(w=p(64), wld=40, ws_bytes=0), L.MTX_ERR_ARG, "workspace"),
    (dict(w=p(64), wld=40, ws=None), L.MTX_ERR_ARG, "workspace"),
])
def test_decode_checks(over, code, frag):
    rc, msg = decode(over)
    assert (rc, frag in msg) == (code, True), msg


@pytest.mark.parametrize("over,code,frag", [
    (dict(cache=3), L.MTX_ERR_DTYPE, "cache"),
    (dict(keep=0, recent=0), L.MTX_ERR_SHAPE, "keep"),
    (dict(recent=17), L.MTX_ERR_SHAPE, "recent"),
    (dict(recent=-1), L.MTX_ERR_SHAPE, "recent"),
    (dict(keep=17), L.MTX_ERR_SHAPE, "hold"),
    (dict(to_pages=0), L.MTX_ERR_SHAPE, "hold"),
    (dict(w=None), L.MTX_ERR_ARG, "null"),
    (dict(slots=None), L.MTX_ERR_ARG, "null"),
    (dict(wld=39), L.MTX_ERR_ARG, "40"),
    (dict(w_out=p(256)), L.MTX_ERR_ARG, "others"),
    (dict(lengths_out=p(128)), L.MTX_ERR_ARG, "others"),
    (dict(to=p(64)), L.MTX_ERR_ARG, "others"),
])
def test_evict_checks(over, code, frag):
    rc, msg = evict(over)
    assert (rc, frag in msg) == (code, True), msg


def test_workspace_queries():
    f = L.lib().mtx_attn_decode_paged_workspace_bytes
    assert f(0, 8, 4, 64, 8, 5, 0) == 0
    assert f(2, 8, 4, 64, 8, 5, 1) >= 0


def forward(over):
    return call("mtx_token_logprobs", dict(
        dtype=0, rows=4, V=100, x=p(16), ld=100, tok=p(32), scale=1.0, lp=p(64), lse=p(64), ent=p(64), top=5, ids=p(64),
        tops=p(64), ws=p(1024), ws_bytes=BIG, stream=None), over)


def backward(over):
    return call("mtx_token_logprobs_bwd", dict(
        dtype=0, rows=4, V=100, x=p(16), ld=100, tok=p(32), lse=p(64), ent=p(64), g=p(64), gh=p(64), scale=1.0,
        dx=p(1024), ldd=100, accumulate=0, stream=None), over)


@pytest.mark.parametrize("fn", [forward, backward])
@pytest.mark.parametrize("over,code,frag", [
    (dict(dtype=9), L.MTX_ERR_DTYPE, "dtype"),
    (dict(rows=0), L.MTX_ERR_SHAPE, "rows"),
    (dict(V=0), L.MTX_ERR_SHAPE, "rows"),
    (dict(x=None), L.MTX_ERR_ARG, "null"),
    (dict(tok=None), L.MTX_ERR_ARG, "null"),
    (dict(x=p(18)), L.MTX_ERR_ARG, "aligned"),
    (dict(ld=99), L.MTX_ERR_ARG, "row stride"),
    (dict(scale=-1.0), L.MTX_ERR_ARG, "scale"),
    (dict(scale=float("inf")), L.MTX_ERR_ARG, "scale"),
    (dict(lse=None), L.MTX_ERR_ARG, "null"),
    (dict(ent=None), L.MTX_ERR_ARG, "null"),
])
def test_logprobs_checks(fn, over, code, frag):
    rc, msg = fn(over)
    assert (rc, frag in msg) == (code, True), msg


@pytest.mark.parametrize("over,code,frag", [
    (dict(top=65), L.MTX_ERR_SHAPE, "top"),
    (dict(top=-1), L.MTX_ERR_SHAPE, "top"),
    (dict(V=4, top=5), L.MTX_ERR_SHAPE, "top"),
    (dict(ids=None), L.MTX_ERR_ARG, "null"),
    (dict(tops=None), L.MTX_ERR_ARG, "null"),
    (dict(lp=None), L.MTX_ERR_ARG, "null"),
])
def test_logprobs_forward_checks(over, code, frag):
    rc, msg = forward(over)
    assert (rc, frag in msg) == (code, True), msg


@pytest.mark.parametrize("over,frag", [(dict(dx=None), "null"), (dict(dx=p(1026)), "row stride"),
                                       (dict(ldd=99), "row stride")])
def test_logprobs_backward_checks(over, frag):
    rc, msg = backward(over)
    assert rc == L.MTX_ERR_ARG and frag in msg


class OnGpu:
    """What the wrappers look at of a tensor on GPU `index`."""

    is_cuda = True

    def __init__(self, shape, dtype="float32", index=0):
        self.shape, self.dtype, self.index = shape, dtype, index

    def stride(self, d=None):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return tuple(s) if d is None else s[d]

    def get_device(self):
        return self.index

    def data_ptr(self):
        raise AssertionError("launched")


@pytest.mark.parametrize("elsewhere", range(7))
def test_arrays_of_another_gpu_are_refused(monkeypatch, elsewhere):
    from minitorch_amd import kernels as K

    monkeypatch.setattr(K.dev, "device", lambda: 0)
    monkeypatch.setattr(K.dev, "SEVERAL", True)
    monkeypatch.setattr(K.dev, "empty_buf", lambda shape, dtype="float32": OnGpu(tuple(shape), dtype))
    gpu = [int(i == elsewhere) for i in range(9)]
    pool, head = (10, 4, 8, 64), (2, 4, 1, 64)
    kp, vp = OnGpu(pool, index=gpu[0]), OnGpu(pool, index=gpu[1])
    table, lengths = OnGpu((2, 5), "int32", gpu[2]), OnGpu((2,), "int32", gpu[3])
    rows = [OnGpu(head, index=gpu[4]), OnGpu(head, index=gpu[5])]
    counts = OnGpu((2,), "int32", gpu[6])
    with pytest.raises(ValueError, match="GPU 0"):
        K.kv_append_paged(*rows, kp, vp, table, lengths, counts)
    w = OnGpu((2, 4, 40), index=gpu[6])
    with pytest.raises(ValueError, match="GPU 0"):
        K.attn_decode_paged(rows[0], kp, vp, table, lengths, 0.125, out=rows[1], weights=w)
    to, w_out = OnGpu((2, 2), "int32", gpu[4]), OnGpu((2, 4, 40), index=gpu[5])
    with pytest.raises(ValueError, match="GPU 0"):
        K.kv_evict_paged(kp, vp, table, lengths, w, to, 16, 4, weights_out=w_out)
    x, tok = OnGpu((6, 50), index=gpu[0]), OnGpu((6,), "int64", gpu[1])
    lp, h, lse = (OnGpu((6,), index=gpu[i]) for i in (2, 3, 4))
    ids, tops = OnGpu((6, 3), "int64", gpu[5]), OnGpu((6, 3), index=gpu[6])
    with pytest.raises(ValueError, match="GPU 0"):
        K.token_logprobs(x, tok, 3, 1.0, lp, h, lse, ids, tops)
    g = [OnGpu((6,), index=gpu[i]) for i in (2, 5)]
    with pytest.raises(ValueError, match="GPU 0"):
        K.token_logprobs_bwd(x, tok, lse, h, *g, dlogits=OnGpu((6, 50), index=gpu[6]))


def test_arrays_of_the_librarys_gpu_are_not(monkeypatch):
    from minitorch_amd import kernels as K

    monkeypatch.setattr(K.dev, "device", lambda: 0)
    monkeypatch.setattr(K.dev, "SEVERAL", True)
    x, tok = OnGpu((6, 50)), OnGpu((6,), "int64")
    v = [OnGpu((6,)) for _ in range(3)]
    with pytest.raises(AssertionError, match="launched"):
        K.token_logprobs(x, tok, 0, 1.0, *v, OnGpu((6, 0), "int64"), OnGpu((6, 0)))


@pytest.mark.parametrize("fn", [forward, backward])
@pytest.mark.parametrize("scale", [1e-28, 1e-40, 1.01e38, 3e38])
def test_scales_that_hidden_logits_or_fp32_do_not_stand(fn, scale):
    """Logits far below the maximum are taken for 1e30 below it, which has to
    have probability 0; the scale times log2 e has to be finite."""
    rc, msg = fn(dict(scale=scale))
    assert rc == L.MTX_ERR_ARG and "scale" in msg
