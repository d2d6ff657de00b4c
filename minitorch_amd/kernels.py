"""Thin Python wrappers over the libmtx_hip entry points.

Each function takes device arrays (``device.DevBuf``: pointer, shape,
element strides, dtype), validates shapes on the host, calls the C ABI on the
current HIP stream and returns the outputs, allocating those not given with
the library's caching allocator.  Errors raise ``ValueError`` (bad
arguments, found before any HIP call) or ``MtxError`` (HIP failure).
"""
from __future__ import annotations

import ctypes
import functools
import sys

import numpy as np

from . import _lib as L
from . import device as dev
from .device import dtype_name as _dt


def _need_cuda(*ts):
    for t in ts:
        if not getattr(t, "is_cuda", False) or not hasattr(t, "data_ptr"):
            raise ValueError("minitorch_amd kernels take device arrays")


def _bhtd(name, t):
    if t.dim() != 4:
        raise ValueError(f"{name}: expected a (B, H, T, D) tensor, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last (d) dimension must be contiguous")


def pack3(srcs, dst):
    """dst (rows, 3*cols) = [s0 | s1 | s2] for three contiguous fp32 (rows,
    cols) tensors (mtx_pack3_f32)."""
    s0, s1, s2 = srcs
    rows, cols = s0.shape
    _need_cuda(s0, s1, s2, dst)
    for t in (s0, s1, s2):
        if tuple(t.shape) != (rows, cols) or not t.is_contiguous() or _dt(t) != "float32":
            raise ValueError("pack3: sources must be contiguous fp32 tensors of one shape")
    if tuple(dst.shape) != (rows, 3 * cols) or not dst.is_contiguous() or _dt(dst) != "float32":
        raise ValueError(f"pack3: dst must be contiguous fp32 ({rows}, {3 * cols})")
    L.call("mtx_pack3_f32", L.ptr(s0), L.ptr(s1), L.ptr(s2), rows, cols, L.ptr(dst),
           L.stream_handle())
    return dst


def unpack3(src, dsts, accumulate=(False, False, False)):
    """d_b (rows, cols) (+)= src[:, b*cols:(b+1)*cols] (mtx_unpack3_f32)."""
    d0, d1, d2 = dsts
    rows, cols = d0.shape
    _need_cuda(src, d0, d1, d2)
    for t in (d0, d1, d2):
        if tuple(t.shape) != (rows, cols) or not t.is_contiguous() or _dt(t) != "float32":
            raise ValueError("unpack3: targets must be contiguous fp32 tensors of one shape")
    if tuple(src.shape) != (rows, 3 * cols) or not src.is_contiguous() or _dt(src) != "float32":
        raise ValueError(f"unpack3: src must be contiguous fp32 ({rows}, {3 * cols})")
    mask = sum(1 << i for i, a in enumerate(accumulate) if a)
    L.call("mtx_unpack3_f32", L.ptr(src), rows, cols, L.ptr(d0), L.ptr(d1), L.ptr(d2), mask,
           L.stream_handle())


def _check_keep(keep, B, H, Tq, Tk):
    """A dropout keep-mask as the kernels take it: contiguous uint8
    (B, H, Tq, ld) with ld >= Tk, ld % 4 == 0 (nonzero = kept)."""
    if _dt(keep) != "uint8" or not keep.is_contiguous() or keep.dim() != 4:
        raise ValueError("keep must be a contiguous uint8 (B,H,Tq,ld) tensor")
    if tuple(keep.shape[:3]) != (B, H, Tq) or keep.shape[3] < Tk or keep.shape[3] % 4:
        raise ValueError(f"keep shape {tuple(keep.shape)} does not fit (B,H,Tq)={(B, H, Tq)}, Tk={Tk}")
    if not getattr(keep, "is_cuda", False):
        raise ValueError("keep must be a device array")
    return keep.shape[3]


def keep_ld(Tk: int) -> int:
    """Row stride (bytes) of a keep-mask for Tk keys."""
    return (Tk + 3) // 4 * 4


def dropout_keep_philox(shape, p: float, seed: int, offset: int, out=None, subsequence: int = 0, base=None):
    """Keep-mask (B, H, Tq, keep_ld(Tk)) uint8 for dropout probability p, from
    the device Philox4x32-10 generator (mtx_dropout_keep): element e of the
    logical (B*H*Tq, Tk) array uses output word e % 4 of counter offset + e // 4
    in the generator's `subsequence`.  base: a device int64 (1,) array that is
    added to offset when the kernel runs.  Returns (mask, next offset)."""
    B, H, Tq, Tk = (int(x) for x in shape)
    ld = keep_ld(Tk)
    if base is not None:
        _on_device(base)
        _vector("base", _spec(base), 1, "int64")
    if out is None:
        out = dev.empty_buf((B, H, Tq, ld), "uint8").fill_(0)
    rows = B * H * Tq
    _int32(Tk=Tk)
    L.call("mtx_dropout_keep", L.ptr(out), rows, Tk, ld, float(p), int(seed) & (2**64 - 1),
           int(offset) & (2**64 - 1), int(subsequence) & (2**32 - 1), _ptr(base), L.stream_handle())
    return out, offset + (rows * Tk + 3) // 4


def attn_fwd(q, k, v, scale: float, causal: bool = True, out=None, lse=None, keep=None,
             keep_scale: float = 1.0):
    """Fused attention forward.  q: (B,H,Tq,D), k/v: (B,H,Tk,D), fp32 or bf16,
    any strides with a contiguous last dim.  Returns (out, lse) with out like q
    and lse fp32 (B,H,Tq).  keep: optional dropout keep-mask (see
    _check_keep); then out = (P * keep * keep_scale) @ v."""
    _need_cuda(q, k, v)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _bhtd(name, t)
    B, H, Tq, D = q.shape
    Tk = k.shape[2]
    if k.shape != (B, H, Tk, D) or v.shape != (B, H, Tk, D):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if not (_dt(q) == _dt(k) == _dt(v)):
        raise ValueError("q, k, v must share a dtype")
    if out is None:
        out = dev.empty_buf((B, H, Tq, D), _dt(q))
    if lse is None:
        lse = dev.empty_buf((B, H, Tq), "float32")
    _bhtd("out", out)
    if not lse.is_contiguous() or tuple(lse.shape) != (B, H, Tq) or _dt(lse) != "float32":
        raise ValueError("lse must be a contiguous fp32 (B,H,Tq) tensor")
    if keep is not None:
        ld = _check_keep(keep, B, H, Tq, Tk)
        L.call("mtx_attn_fwd_dropout", L.dtype_code(q), B, H, Tq, Tk, D,
               L.ptr(q), L.strides(q), L.ptr(k), L.strides(k), L.ptr(v), L.strides(v),
               L.ptr(out), L.strides(out), L.ptr(lse), float(scale), int(bool(causal)),
               L.ptr(keep), ld, float(keep_scale), L.stream_handle())
        return out, lse
    L.call("mtx_attn_fwd", L.dtype_code(q), B, H, Tq, Tk, D,
           L.ptr(q), L.strides(q), L.ptr(k), L.strides(k), L.ptr(v), L.strides(v),
           L.ptr(out), L.strides(out), L.ptr(lse), float(scale), int(bool(causal)),
           L.stream_handle())
    return out, lse


def attn_decode(q, k, v, scale: float, out=None, lse=None, lengths=None):
    """Decode-step attention: q (B,H,1,D) against k/v (B,H,L,D) (any strides
    with a contiguous last dim, e.g. head views of (B,T,C) caches).  lengths:
    optional int32 device tensor (B,): sequence b uses its first lengths[b]
    keys.  Returns (out (B,H,1,D) like q, lse fp32 (B,H) or None)."""
    _need_cuda(q, k, v)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _bhtd(name, t)
    B, H, Tq, D = q.shape
    Lk = k.shape[2]
    if Tq != 1 or k.shape != (B, H, Lk, D) or v.shape != (B, H, Lk, D):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if not (_dt(q) == _dt(k) == _dt(v)):
        raise ValueError("q, k, v must share a dtype")
    if out is None:
        out = dev.empty_buf((B, H, 1, D), _dt(q))
    _bhtd("out", out)
    if lse is not None and (not lse.is_contiguous() or tuple(lse.shape) != (B, H) or _dt(lse) != "float32"):
        raise ValueError("lse must be a contiguous fp32 (B,H) tensor")
    if lengths is not None and (_dt(lengths) != "int32" or tuple(lengths.shape) != (B,)
                                or not lengths.is_contiguous() or not lengths.is_cuda):
        raise ValueError("lengths must be a contiguous int32 device tensor of shape (B,)")
    L.call("mtx_attn_decode", L.dtype_code(q), B, H, Lk, D,
           L.ptr(q), L.strides(q), L.ptr(k), L.strides(k), L.ptr(v), L.strides(v),
           L.ptr(out), L.strides(out), L.ptr(lse) if lse is not None else None,
           L.ptr(lengths) if lengths is not None else None, float(scale),
           L.stream_handle())
    return out, lse


# ---------------------------------------------------------------------------
# keys and values in pages
# ---------------------------------------------------------------------------

# A decode step makes many small calls, so what a wrapper checks and derives of
# its operands' specs -- (shape, strides, dtype) -- is kept per combination of them
# (the cached *_plan functions, which never see an address); a call then only
# passes pointers.  The specs of operands that are always there are formed in
# place: a function call each would cost as much as the rest.

def _spec(t):
    """The spec of a device array; None for None."""
    if t is None:
        return None
    if not t.is_cuda:
        _need_cuda(t)
    return t.shape, t.stride(), t.dtype


def _on_device(*ts):
    """Raises unless every operand is a device array."""
    for t in ts:
        if not getattr(t, "is_cuda", False):
            raise ValueError("minitorch_amd kernels take device arrays")


def _on_gpu0(*ts):
    """Where there are several GPUs: raises unless every operand (None: not
    there) lies on the library's and the thread's launches go there."""
    for t in ts:
        if getattr(t, "get_device", int)() != 0:
            raise ValueError("minitorch_amd kernels take arrays of GPU 0")
    torch = sys.modules.get("torch")
    if torch is not None and torch.cuda.is_initialized() and torch.cuda.current_device() != 0:
        raise ValueError("minitorch_amd kernels run on GPU 0, which is not the current device")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ints(*xs):
    """ints as the C ints of an argument list, converted once."""
    return tuple(ctypes.c_int(x) for x in xs)


def _longs(*xs):
    return tuple(ctypes.c_int64(x) for x in xs)


def _packed(shape, strides):
    """Whether strides are C order's (those of dimensions of 1 do not matter)."""
    acc = 1
    for n, st in zip(shape[::-1], strides[::-1]):
        if n != 1 and st != acc:
            return False
        acc *= n
    return True


def _vector(name, spec, n, dtype):
    if spec is not None and (_dt(spec[2]) != dtype or tuple(spec[0]) != (n,) or not _packed(spec[0], spec[1])):
        raise ValueError(f"{name} must be contiguous {dtype} ({n},)")


def _view4(name, spec):
    """(shape, stride array, dtype) of a 4-d view with a contiguous last axis."""
    shape, strides, dtype = spec
    if len(shape) != 4 or strides[3] != 1:
        raise ValueError(f"{name}: expected a 4-d view with a contiguous last (d) axis, got shape {tuple(shape)}, "
                         f"strides {tuple(strides)}")
    return tuple(shape), L.stride_array(tuple(strides)), _dt(dtype)


def _paged(k_pages, v_pages, table, lengths):
    """Checks a paged cache's specs: two (n_pages, Hkv, page, D) views of one
    dtype, an int32 (B, max_pages) table with contiguous rows and int32 (B,)
    lengths.  Returns (shape, dtype, the views' strides, B, table row stride,
    max_pages)."""
    shape, ks, dtype = _view4("k_pages", k_pages)
    vshape, vs, vdtype = _view4("v_pages", v_pages)
    if shape != vshape or dtype != vdtype:
        raise ValueError("k_pages and v_pages must be (n_pages, Hkv, page, D) views of one shape and dtype")
    B, width, ld = _table("table", table)
    _vector("lengths", lengths, B, "int32")
    return shape, dtype, ks, vs, B, ld, width


def _table(name, spec, B=None):
    shape, strides, dtype = spec
    if _dt(dtype) != "int32" or len(shape) != 2 or strides[1] != 1 or (B is not None and shape[0] != B):
        raise ValueError(f"{name} must be int32 ({'B' if B is None else B}, pages) with contiguous rows")
    return shape[0], shape[1], strides[0]


def _row_weights(name, spec, B, Hkv, cap, like=None):
    """Checks weights of cached rows: contiguous fp32 (B, Hkv, >= cap)."""
    shape, strides, dtype = spec
    if _dt(dtype) != "float32" or len(shape) != 3 or tuple(shape[:2]) != (B, Hkv) or shape[2] < cap \
            or not _packed(shape, strides) or (like is not None and shape[2] != like):
        raise ValueError(f"{name} must be contiguous fp32 ({B}, {Hkv}, {like or f'>= {cap}'})")
    return shape[2]


_CODES = {"float32": L.MTX_F32, "bfloat16": L.MTX_BF16}


def _code(dtype):
    if dtype not in _CODES:
        raise ValueError(f"unsupported dtype {dtype} (float32 or bfloat16)")
    return _CODES[dtype]


@functools.lru_cache(maxsize=512)
def _append_plan(k, v, k_pages, v_pages, table, lengths, counts):
    (n_pages, Hkv, page, D), cache, kps, vps, B, ld, width = _paged(k_pages, v_pages, table, lengths)
    kshape, ks, kd = _view4("k", k)
    vshape, vs, vd = _view4("v", v)
    T = kshape[2]
    if kshape != (B, Hkv, T, D) or vshape != kshape or kd != vd:
        raise ValueError(f"k and v must be ({B}, {Hkv}, T, {D}) of one dtype (got {kshape}, {vshape})")
    _vector("counts", counts, B, "int32")
    dev.device()
    return (_code(kd), _code(cache), B, T, Hkv, D), (ks, vs), (n_pages, page), (kps, vps), (ld, width)


def kv_append_paged(k, v, k_pages, v_pages, table, lengths, counts=None):
    """Write the keys and values of T new tokens per sequence, k and v
    (B, Hkv, T, D) views, to the end of its pages (mtx_kv_append_paged).
    lengths (B,) counts them already; counts (int32 (B,)): sequence b appends
    only its first counts[b] rows.  fp32 rows may go to a bf16 pool."""
    if not (k.is_cuda and v.is_cuda and k_pages.is_cuda and v_pages.is_cuda and table.is_cuda and lengths.is_cuda):
        _on_device(k, v, k_pages, v_pages, table, lengths)
    sizes, (ks, vs), (n, page), (kps, vps), (ld, width) = _append_plan(
        (k.shape, k.stride(), k.dtype), (v.shape, v.stride(), v.dtype),
        (k_pages.shape, k_pages.stride(), k_pages.dtype), (v_pages.shape, v_pages.stride(), v_pages.dtype),
        (table.shape, table.stride(), table.dtype), (lengths.shape, lengths.stride(), lengths.dtype), _spec(counts))
    if dev.SEVERAL:
        _on_gpu0(k, v, k_pages, v_pages, table, lengths, counts)
    L.call("mtx_kv_append_paged", *sizes, k.data_ptr(), ks, v.data_ptr(), vs, n, page, k_pages.data_ptr(), kps,
           v_pages.data_ptr(), vps, table.data_ptr(), ld, width, lengths.data_ptr(), _ptr(counts), L.stream_handle())


@functools.lru_cache(maxsize=512)
def _decode_paged_plan(q, k_pages, v_pages, table, lengths, out, lse, weights, weights_in):
    (n_pages, Hkv, page, D), cache, kps, vps, B, ld, width = _paged(k_pages, v_pages, table, lengths)
    qshape, qs, qd = _view4("q", q)
    H = qshape[1]
    if qshape != (B, H, 1, D):
        raise ValueError(f"q must be ({B}, H, 1, {D}) (got {qshape})")
    oshape, os, od = _view4("out", out)
    if oshape != qshape or od != qd:
        raise ValueError("out must have q's shape and dtype")
    if lse is not None and (_dt(lse[2]) != "float32" or tuple(lse[0]) != (B, H) or not _packed(*lse[:2])):
        raise ValueError("lse must be a contiguous fp32 (B,H) tensor")
    wld = 0
    if weights is not None:
        wld = _row_weights("weights", weights, B, Hkv, width * page)
        if weights_in is not None:
            _row_weights("weights_in", weights_in, B, Hkv, width * page, wld)
    elif weights_in is not None:
        raise ValueError("weights_in without weights")
    ws = L.lib().mtx_attn_decode_paged_workspace_bytes(B, H, Hkv, D, page, width, int(weights is not None))
    dev.device()
    return (_ints(_code(qd), _code(cache), B, H, Hkv, D), (qs, os), (*_longs(n_pages), *_ints(page)), (kps, vps),
            (*_longs(ld), *_ints(width)), *_longs(wld), ws)


def attn_decode_paged(q, k_pages, v_pages, table, lengths, scale: float, out=None, lse=None, weights=None,
                      weights_in=None):
    """Attention of one new token per sequence over its pages
    (mtx_attn_decode_paged): q (B, H, 1, D), H a multiple of the pool's Hkv,
    fp32 or bf16 over a pool of the same dtype or fp32 over bf16.  weights
    (B, Hkv, >= max_pages * page) fp32: receives weights_in (0 without it; it
    may be weights itself) plus the attention each cached row got.  Returns
    (out like q, lse or None)."""
    if not (q.is_cuda and k_pages.is_cuda and v_pages.is_cuda and table.is_cuda and lengths.is_cuda):
        _on_device(q, k_pages, v_pages, table, lengths)
    if out is None:
        out = dev.empty_buf(q.shape, _dt(q))
    sizes, (qs, os), (n, page), (kps, vps), (ld, width), wld, ws_bytes = _decode_paged_plan(
        (q.shape, q.stride(), q.dtype), (k_pages.shape, k_pages.stride(), k_pages.dtype),
        (v_pages.shape, v_pages.stride(), v_pages.dtype), (table.shape, table.stride(), table.dtype),
        (lengths.shape, lengths.stride(), lengths.dtype), _spec(out), _spec(lse), _spec(weights), _spec(weights_in))
    if dev.SEVERAL:
        _on_gpu0(q, k_pages, v_pages, table, lengths, out, lse, weights, weights_in)
    ws = dev.empty_buf((ws_bytes,), "uint8") if ws_bytes else None
    L.call("mtx_attn_decode_paged", *sizes, q.data_ptr(), qs, n, page, k_pages.data_ptr(), kps, v_pages.data_ptr(),
           vps, table.data_ptr(), ld, width, lengths.data_ptr(), out.data_ptr(), os, _ptr(lse), _ptr(weights_in),
           _ptr(weights), wld, _ptr(ws), ws_bytes, float(scale), L.stream_handle())
    return out, lse


@functools.lru_cache(maxsize=512)
def _evict_plan(k_pages, v_pages, table, lengths, weights, to_table, keep, lengths_out, weights_out, slots):
    (n_pages, Hkv, page, D), cache, kps, vps, B, ld, width = _paged(k_pages, v_pages, table, lengths)
    wld = _row_weights("weights", weights, B, Hkv, width * page)
    _, to_pages, to_ld = _table("to_table", to_table, B)
    _vector("lengths_out", lengths_out, B, "int32")
    _row_weights("weights_out", weights_out, B, Hkv, width * page, wld)
    if _dt(slots[2]) != "int32" or tuple(slots[0]) != (B, Hkv, keep) or not _packed(*slots[:2]):
        raise ValueError(f"slots must be contiguous int32 ({B}, {Hkv}, {keep})")
    dev.device()
    return (_code(cache), B, Hkv, D, n_pages, page), (kps, vps), (ld, width), wld, (to_ld, to_pages)


def kv_evict_paged(k_pages, v_pages, table, lengths, weights, to_table, keep: int, recent: int, lengths_out=None,
                   weights_out=None, slots=None):
    """Cut each sequence and K/V head down to its last `recent` rows and the
    keep - recent others of greatest weight, written in order to the pages of
    to_table (mtx_kv_evict_paged): int32 (B, to_pages), pages of the same pool
    that no table of the call reads.  weights as attn_decode_paged accumulates
    them.  Returns (lengths_out (B,), weights_out like weights, slots
    (B, Hkv, keep) int32: the rows kept, then -1).  Columns of weights_out behind
    the table's rows are 0 if it is not given, else left as they were."""
    keep = int(keep)
    if keep < 1:
        raise ValueError("keep must be at least 1")
    if lengths_out is None:
        lengths_out = dev.empty_buf(lengths.shape, "int32")
    made = weights_out is None
    if made:
        weights_out = dev.empty_buf(weights.shape, "float32")
    if slots is None:
        slots = dev.empty_buf((table.shape[0], k_pages.shape[1], keep), "int32")
    sizes, (kps, vps), (ld, width), wld, (to_ld, to_pages) = _evict_plan(
        _spec(k_pages), _spec(v_pages), _spec(table), _spec(lengths), _spec(weights), _spec(to_table), keep,
        _spec(lengths_out), _spec(weights_out), _spec(slots))
    if dev.SEVERAL:
        _on_gpu0(k_pages, v_pages, table, lengths, weights, to_table, lengths_out, weights_out, slots)
    if made and wld > width * k_pages.shape[2]:
        weights_out.fill_(0.0)
    L.call("mtx_kv_evict_paged", *sizes, k_pages.data_ptr(), kps, v_pages.data_ptr(), vps, table.data_ptr(), ld,
           width, lengths.data_ptr(), weights.data_ptr(), wld, to_table.data_ptr(), to_ld, to_pages, keep,
           int(recent), lengths_out.data_ptr(), weights_out.data_ptr(), slots.data_ptr(), L.stream_handle())
    return lengths_out, weights_out, slots


DECODE_STEP_WIDTHS = (128, 256, 384, 512)
_DECODE_LAYER_KEYS = ("ln1_gamma", "ln1_beta", "w_qkv", "b_qkv", "w_out", "b_out", "ln2_gamma", "ln2_beta",
                      "w_fc1", "b_fc1", "w_fc2", "b_fc2", "k_cache", "v_cache")


def decode_step_fits(n_layer, C, n_head, F, V, Tmax):
    """Whether mtx_decode_step_f32 runs the model: head size 64 with C in
    {128, 256, 384, 512}, MLP width F = 4C, V <= 256, up to 16 blocks and
    1024 cache rows."""
    return (C in DECODE_STEP_WIDTHS and C == 64 * n_head and F == 4 * C
            and 1 <= V <= 256 and 1 <= n_layer <= 16 and 1 <= Tmax <= 1024)


class DecodeStep:
    """A GPT's greedy decode step as one persistent, cooperative launch
    (mtx_decode_step_f32): embeddings, every block, ln_f, lm_head and the
    pick, with grid-wide barriers between stages.

    layers: one dict per block of fp32 device arrays, contiguous, weights
    (in, out): ln1_gamma, ln1_beta, w_qkv (C, 3C) [q | k | v], b_qkv, w_out
    (C, C), b_out, ln2_gamma, ln2_beta, w_fc1 (C, F), b_fc1, w_fc2 (F, C),
    b_fc2, k_cache and v_cache (B, Tmax, C), plus ln1_eps and ln2_eps
    floats.  tok_emb (n_tok, C), pos_emb (n_pos, C), lnf = (gamma, beta,
    eps), w_head (C, V), b_head (V,).  The workspace (barrier words, residual
    rows, partial products) is allocated and zeroed here; the steps of one
    DecodeStep run in order on one stream."""

    def __init__(self, layers, tok_emb, pos_emb, lnf, w_head, b_head, B, Tmax):
        C = tok_emb.shape[1]
        F = layers[0]["w_fc1"].shape[1]
        V = w_head.shape[1]
        H = C // 64
        if not decode_step_fits(len(layers), C, H, F, V, Tmax):
            raise ValueError("decode_step: model outside the persistent step's limits")
        arrays = [tok_emb, pos_emb, lnf[0], lnf[1], w_head, b_head]
        for y in layers:
            arrays += [y[k] for k in _DECODE_LAYER_KEYS]
        for t in arrays:
            _need_cuda(t)
            if _dt(t) != "float32" or not t.is_contiguous():
                raise ValueError("decode_step: model arrays must be contiguous fp32 device arrays")
        shapes = {"w_qkv": (C, 3 * C), "b_qkv": (3 * C,), "w_out": (C, C), "b_out": (C,), "w_fc1": (C, F),
                  "b_fc1": (F,), "w_fc2": (F, C), "b_fc2": (C,), "ln1_gamma": (C,), "ln1_beta": (C,),
                  "ln2_gamma": (C,), "ln2_beta": (C,), "k_cache": (B, Tmax, C), "v_cache": (B, Tmax, C)}
        for i, y in enumerate(layers):
            for k, s in shapes.items():
                if tuple(y[k].shape) != s:
                    raise ValueError(f"decode_step: layer {i} {k} has shape {tuple(y[k].shape)}, expected {s}")
        if tuple(w_head.shape) != (C, V) or tuple(b_head.shape) != (V,) or pos_emb.shape[1] != C:
            raise ValueError("decode_step: head or embedding shapes do not match")
        self.B, self.C, self.Tmax, self.V = B, C, Tmax, V
        self._arrays = arrays  # kept alive: the structs below hold their addresses
        self._layers = (L.DecodeLayer * len(layers))()
        for i, y in enumerate(layers):
            for k in _DECODE_LAYER_KEYS:
                setattr(self._layers[i], k, y[k].data_ptr())
            self._layers[i].ln1_eps = float(y["ln1_eps"])
            self._layers[i].ln2_eps = float(y["ln2_eps"])
        m = L.DecodeModel()
        m.n_layer, m.B, m.C, m.n_head, m.F, m.V, m.Tmax = len(layers), B, C, H, F, V, Tmax
        m.tok_emb, m.n_tok = tok_emb.data_ptr(), tok_emb.shape[0]
        m.pos_emb, m.n_pos = pos_emb.data_ptr(), pos_emb.shape[0]
        m.layers = self._layers
        m.lnf_gamma, m.lnf_beta, m.lnf_eps = lnf[0].data_ptr(), lnf[1].data_ptr(), float(lnf[2])
        m.w_head, m.b_head = w_head.data_ptr(), b_head.data_ptr()
        self._model = m
        nbytes = L.lib().mtx_decode_step_workspace_bytes(B, C, H, F)
        self.workspace = dev.zeros(((nbytes + 3) // 4,), "int32").t
        self._ws_bytes = self.workspace.numel() * 4

    def __call__(self, cur, ids, lengths, pos, margins=None, t_base=0, wait_limit_us=0, steps=1):
        """`steps` token steps in one launch.  A step reads cur (B,) int64
        and pos (1,) int64, appends to the caches at row lengths[b] - 1,
        writes the pick to cur and ids (Tmax, B) at row lengths[b], the top-2
        margin to margins (n, B) at row lengths[b] - t_base, then lengths +=
        1 and pos += 1.  wait_limit_us bounds each grid-wide wait (0: the
        library's 2 s; negative: every wait fails, for tests of the failure
        path)."""
        B = self.B
        _need_cuda(cur, ids, lengths, pos)
        if _dt(cur) != "int64" or cur.numel() != B or not cur.is_contiguous():
            raise ValueError("decode_step: cur must be contiguous int64 (B,)")
        if _dt(ids) != "int64" or ids.dim() != 2 or ids.shape[1] != B or not ids.is_contiguous():
            raise ValueError("decode_step: ids must be contiguous int64 (Tmax, B)")
        if _dt(lengths) != "int32" or lengths.numel() != B or not lengths.is_contiguous():
            raise ValueError("decode_step: lengths must be contiguous int32 (B,)")
        if _dt(pos) != "int64" or pos.numel() < 1:
            raise ValueError("decode_step: pos must be int64")
        if margins is not None and (_dt(margins) != "float32" or margins.dim() != 2 or margins.shape[1] != B
                                    or not margins.is_contiguous()):
            raise ValueError("decode_step: margins must be contiguous fp32 (n, B)")
        L.call("mtx_decode_step_f32", ctypes.addressof(self._model), int(steps), L.ptr(cur), L.ptr(ids),
               L.ptr(margins) if margins is not None else None, int(t_base),
               margins.shape[0] if margins is not None else 0, L.ptr(lengths), L.ptr(pos),
               L.ptr(self.workspace), self._ws_bytes, int(wait_limit_us), L.stream_handle())

    def check(self):
        """Synchronise and raise MtxError if a step's grid-wide wait ran out
        (that step's results are incomplete; later steps did nothing)."""
        L.call("mtx_decode_step_status", L.ptr(self.workspace), L.stream_handle())

    def reset(self):
        """Clear the barrier words and the error word."""
        L.call("mtx_decode_step_reset", L.ptr(self.workspace), L.stream_handle())


QKV_ATTN_MAX_C, QKV_ATTN_MAX_T = 1024, 2048


def qkv_attn_fits(H, D, Tmax):
    """True when mtx_decode_qkv_attn_f32 takes heads of size D, H*D columns
    and caches of Tmax rows."""
    return D in (64, 128) and H * D <= QKV_ATTN_MAX_C and 1 <= Tmax <= QKV_ATTN_MAX_T


def _pending_args(pending, ln, rows, C):
    """ctypes arguments (pws, pks, pbias) and (gamma, beta, eps) of the
    pending-update input mode of mtx_decode_qkv_attn_f32 / mtx_head_pick_f32."""
    if ln is None:
        if pending is not None:
            raise ValueError("pending partial products need the LayerNorm (ln)")
        return (None, 0, None), (None, None, 0.0)
    gamma, beta, eps = ln
    if gamma.numel() != C or beta.numel() != C or not (gamma.is_contiguous() and beta.is_contiguous()):
        raise ValueError(f"ln: gamma and beta must be contiguous with {C} elements")
    if C > 1024:
        raise ValueError("the LayerNorm input mode needs rows of at most 1024 values")
    lnargs = (L.ptr(gamma), L.ptr(beta), float(eps))
    if pending is None:
        return (None, 0, None), lnargs
    ws, ks, pbias = pending
    if not 1 <= int(ks) <= 8 or ws.numel() * ws.element_size() < int(ks) * rows * C * 4:
        raise ValueError("pending: 1 to 8 partial products of (rows, C) fp32")
    if pbias is not None and (pbias.numel() != C or not pbias.is_contiguous()):
        raise ValueError(f"pending: bias must be contiguous with {C} elements")
    return (L.ptr(ws), int(ks), L.ptr(pbias) if pbias is not None else None), lnargs


def gemm_partials(a, b, ws=None):
    """mtx_gemm_partials_f32: the K ranges' partial products of a (M, K) @
    b (K, N) into ws ([ks][M][N] fp32; allocated when None).  Returns
    (ws, ks).  Summed in range order they are mtx_gemm_ln_f32's product."""
    import ctypes

    M, Kd = a.shape[-2], a.shape[-1]
    N = b.shape[-1]
    if _dt(a) != "float32" or _dt(b) != "float32" or b.shape[-2] != Kd:
        raise ValueError("gemm_partials: fp32 a (M, K) and b (K, N)")
    nbytes = L.lib().mtx_gemm_ln_workspace_bytes(M, N, Kd)
    if ws is None:
        ws = dev.empty_buf((nbytes // 4,), "float32")
    ks = ctypes.c_int(0)
    L.call("mtx_gemm_partials_f32", int(M), int(N), int(Kd), L.ptr(a), int(a.stride(-2)), int(a.stride(-1)),
           L.ptr(b), int(b.stride(-2)), int(b.stride(-1)), L.ptr(ws), ws.numel() * ws.element_size(),
           ctypes.byref(ks), L.stream_handle())
    return ws, ks.value


def qkv_attn_step(x, w, bias, kc, vc, lengths, n_head, scale, out, pending=None, x_out=None, ln=None):
    """mtx_decode_qkv_attn_f32: one decode step's q/k/v projection and
    attention in one launch.  x (B, C) the input rows, w (C, 3C) and bias
    (3C,) the packed [q | k | v] projection; this step's k and v go to row
    lengths[b] - 1 of the caches kc / vc (B, Tmax, C), and out (B, C)
    receives softmax(scale q k^T) v over each sequence's first lengths[b]
    cached rows, head h in columns h*D .. h*D + D - 1.  Without ln the rows
    of x are the normalised input; with ln = (gamma, beta, eps) they are raw
    residual rows r (plus, with pending = (ws, ks, bias), the previous
    block's pending update r = (sum of the ks partial products + bias) + x,
    written to x_out) and the projection reads LayerNorm(r)."""
    _need_cuda(x, w, kc, vc, lengths, out)
    B, C = x.shape
    H = int(n_head)
    D = C // H
    Bc, Tmax, Ck = kc.shape
    if H * D != C or tuple(w.shape) != (C, 3 * C) or Ck != C or Bc < B or tuple(out.shape) != (B, C):
        raise ValueError("qkv_attn_step: x (B, C), w (C, 3C), caches (>= B, T, C), out (B, C)")
    if tuple(vc.shape) != tuple(kc.shape) or tuple(vc.stride()) != tuple(kc.stride()) or kc.stride(2) != 1:
        raise ValueError("qkv_attn_step: k/v caches must share shape and strides, unit column stride")
    if x.stride(1) != 1 or w.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("qkv_attn_step: x, w and out need unit column strides")
    if bias is not None and (bias.numel() != 3 * C or not bias.is_contiguous()):
        raise ValueError("qkv_attn_step: bias must be contiguous (3C,)")
    if _dt(lengths) != "int32" or lengths.numel() < B or not lengths.is_contiguous():
        raise ValueError("qkv_attn_step: lengths must be contiguous int32 with >= B entries")
    pargs, lnargs = _pending_args(pending, ln, B, C)
    if x_out is not None and (ln is None or tuple(x_out.shape) != (B, C) or x_out.stride(1) != 1):
        raise ValueError("qkv_attn_step: x_out (B, C) with a unit column stride, with ln")
    L.call("mtx_decode_qkv_attn_f32", B, H, D, L.ptr(x), x.stride(0), *pargs,
           L.ptr(x_out) if x_out is not None else None, x_out.stride(0) if x_out is not None else 0, *lnargs,
           L.ptr(w), w.stride(0), L.ptr(bias) if bias is not None else None, L.ptr(kc), L.ptr(vc),
           kc.stride(0), kc.stride(1), Tmax, L.ptr(lengths), float(scale), L.ptr(out), out.stride(0),
           L.stream_handle())
    return out


def argmax_rows(x, idx=None, margin=None):
    """First-maximum index of each row of a fp32 (rows, cols) device tensor
    (np.argmax) and, if `margin` is given, largest - second largest.  idx:
    int64 (rows,) or a strided column view; returns (idx, margin)."""
    _need_cuda(x)
    if _dt(x) != "float32" or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("x must be a fp32 (rows, cols) tensor with contiguous rows")
    rows, cols = x.shape
    if idx is None:
        idx = dev.empty_buf((rows,), "int64")
    if _dt(idx) != "int64" or idx.numel() != rows:
        raise ValueError("idx must be int64 with one entry per row")
    if margin is not None and (_dt(margin) != "float32" or margin.numel() != rows):
        raise ValueError("margin must be fp32 with one entry per row")
    L.call("mtx_argmax_f32", rows, cols, L.ptr(x), x.stride(0), L.ptr(idx), idx.stride(0) if idx.dim() else 1,
           L.ptr(margin) if margin is not None else None, margin.stride(0) if margin is not None else 0,
           L.stream_handle())
    return idx, margin


def kv_append(x, cache, lengths):
    """cache[b, lengths[b] - 1, :] = x[b, 0, :]: x (B, 1, C) fp32, cache
    (B, T, C) fp32 with contiguous rows, lengths int32 device (B,)."""
    _need_cuda(x, cache, lengths)
    B, T, C = cache.shape
    if _dt(x) != "float32" or _dt(cache) != "float32" or tuple(x.shape) != (B, 1, C):
        raise ValueError(f"kv_append: x{tuple(x.shape)} / cache{tuple(cache.shape)} mismatch (fp32 needed)")
    if x.stride(2) != 1 or cache.stride(2) != 1 or _dt(lengths) != "int32" or tuple(lengths.shape) != (B,):
        raise ValueError("kv_append: contiguous rows and int32 lengths (B,) needed")
    L.call("mtx_kv_append_f32", B, C, T, L.ptr(x), x.stride(0), L.ptr(cache), cache.stride(0), cache.stride(1),
           L.ptr(lengths), L.stream_handle())


def decode_advance(lengths, pos=None):
    """lengths += 1 (int32 device (B,)) and pos += 1 (int64 device (1,))."""
    _need_cuda(lengths)
    if _dt(lengths) != "int32" or lengths.dim() != 1 or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 device vector")
    if pos is not None and (_dt(pos) != "int64" or not pos.is_cuda):
        raise ValueError("pos must be an int64 device tensor")
    L.call("mtx_decode_advance", lengths.numel(), L.ptr(lengths), L.ptr(pos) if pos is not None else None,
           L.stream_handle())


def attn_bwd(q, k, v, out, dout, lse, scale: float, causal: bool = True,
             dq=None, dk=None, dv=None, accumulate: bool = False, workspace=None,
             phases: int = L.ATTN_BWD_ALL, keep=None, keep_scale: float = 1.0):
    """Fused attention backward.  Returns fp32 (dq, dk, dv).  With
    accumulate=True the given dq/dk/dv are added to instead of overwritten.
    keep/keep_scale: the forward's dropout mask (all phases only)."""
    _need_cuda(q, k, v, out, dout, lse)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("dout", dout)):
        _bhtd(name, t)
    B, H, Tq, D = q.shape
    Tk = k.shape[2]
    if tuple(out.shape) != tuple(q.shape) or tuple(dout.shape) != tuple(q.shape):
        raise ValueError("out and dout must have q's shape")
    if not (_dt(q) == _dt(k) == _dt(v) == _dt(out) == _dt(dout)):
        raise ValueError("q, k, v, out, dout must share a dtype")
    if dq is None:
        dq = dev.empty_buf((B, H, Tq, D), "float32")
    if dk is None:
        dk = dev.empty_buf((B, H, Tk, D), "float32")
    if dv is None:
        dv = dev.empty_buf((B, H, Tk, D), "float32")
    for name, t, shp in (("dq", dq, (B, H, Tq, D)), ("dk", dk, (B, H, Tk, D)), ("dv", dv, (B, H, Tk, D))):
        if tuple(t.shape) != shp or _dt(t) != "float32":
            raise ValueError(f"{name} must be fp32 with shape {shp}")
        _bhtd(name, t)
    nbytes = L.lib().mtx_attn_bwd_workspace_bytes(B, H, Tq)
    if workspace is None:
        workspace = dev.empty_buf((nbytes,), "uint8")
    if keep is not None:
        if int(phases) != L.ATTN_BWD_ALL:
            raise ValueError("the dropout backward runs all phases")
        ld = _check_keep(keep, B, H, Tq, Tk)
        L.call("mtx_attn_bwd_dropout", L.dtype_code(q), B, H, Tq, Tk, D,
               L.ptr(q), L.strides(q), L.ptr(k), L.strides(k), L.ptr(v), L.strides(v),
               L.ptr(out), L.strides(out), L.ptr(dout), L.strides(dout), L.ptr(lse),
               L.ptr(dq), L.strides(dq), L.ptr(dk), L.strides(dk), L.ptr(dv), L.strides(dv),
               L.ptr(workspace), workspace.numel() * workspace.element_size(),
               float(scale), int(bool(causal)), int(bool(accumulate)), L.ptr(keep), ld,
               float(keep_scale), L.stream_handle())
        return dq, dk, dv
    L.call("mtx_attn_bwd_phase", int(phases), L.dtype_code(q), B, H, Tq, Tk, D,
           L.ptr(q), L.strides(q), L.ptr(k), L.strides(k), L.ptr(v), L.strides(v),
           L.ptr(out), L.strides(out), L.ptr(dout), L.strides(dout), L.ptr(lse),
           L.ptr(dq), L.strides(dq), L.ptr(dk), L.strides(dk), L.ptr(dv), L.strides(dv),
           L.ptr(workspace), workspace.numel() * workspace.element_size(),
           float(scale), int(bool(causal)), int(bool(accumulate)), L.stream_handle())
    return dq, dk, dv


def attn_bwd_noalloc(q, k, v, out, dout, lse, scale: float, causal: bool, dq, dk, dv,
                     accumulate: bool = False):
    """mtx_attn_bwd_noalloc: attn_bwd into caller-given dq/dk/dv with the
    library's fixed device scratch for delta (no allocation of any kind; at
    most ATTN_SCRATCH_BYTES / 4 rows B*H*Tq)."""
    _need_cuda(q, k, v, out, dout, lse, dq, dk, dv)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("dout", dout), ("dq", dq), ("dk", dk),
                    ("dv", dv)):
        _bhtd(name, t)
    B, H, Tq, D = q.shape
    Tk = k.shape[2]
    L.call("mtx_attn_bwd_noalloc", L.dtype_code(q), B, H, Tq, Tk, D,
           L.ptr(q), L.strides(q), L.ptr(k), L.strides(k), L.ptr(v), L.strides(v),
           L.ptr(out), L.strides(out), L.ptr(dout), L.strides(dout), L.ptr(lse),
           L.ptr(dq), L.strides(dq), L.ptr(dk), L.strides(dk), L.ptr(dv), L.strides(dv),
           float(scale), int(bool(causal)), int(bool(accumulate)), L.stream_handle())
    return dq, dk, dv


# ---------------------------------------------------------------------------
# generic elementwise / reductions
# ---------------------------------------------------------------------------

def _i64(seq):
    seq = tuple(map(int, seq))
    return (L.C.c_int64 * max(1, len(seq)))(*seq)


def _bstrides(t, shape):
    """Element strides of `t` broadcast to `shape` (0 on broadcast axes)."""
    nd = len(shape)
    ts, tst = tuple(t.shape), tuple(t.stride())
    pad = nd - len(ts)
    if pad < 0:
        raise ValueError(f"cannot broadcast shape {ts} to {tuple(shape)}")
    if ts == shape:
        return [st if sz != 1 else 0 for sz, st in zip(ts, tst)]
    out = []
    for d in range(nd):
        if d < pad:
            out.append(0)
            continue
        sz = ts[d - pad]
        if sz == shape[d]:
            out.append(tst[d - pad] if sz != 1 else 0)
        elif sz == 1:
            out.append(0)
        else:
            raise ValueError(f"cannot broadcast shape {ts} to {tuple(shape)}")
    return out


def ewise(op: str, out, a=None, b=None, alpha: float = 1.0, beta: float = 0.0, accumulate=False):
    """out (+)= op(a, b), broadcasting a and b to out's shape."""
    shape = tuple(out.shape)
    nd = len(shape)
    if nd > 8:
        raise ValueError("at most 8 dimensions")
    sa = _i64(_bstrides(a, shape)) if a is not None else None
    sb = _i64(_bstrides(b, shape)) if b is not None else None
    L.call("mtx_ewise_f32", L.EW[op], nd, _i64(shape),
           L.ptr(a) if a is not None else None, sa,
           L.ptr(b) if b is not None else None, sb,
           L.ptr(out), _i64(out.stride()), float(alpha), float(beta), int(bool(accumulate)),
           L.stream_handle())
    return out


def fill(out, value: float):
    shape = tuple(out.shape)
    L.call("mtx_ewise_f32", L.EW["FILL"], len(shape), _i64(shape), None, None, None, None,
           L.ptr(out), _i64(out.stride()), float(value), 0.0, 0, L.stream_handle())
    return out


def reduce(a, axes, out, op=L.RED_SUM, alpha: float = 1.0, accumulate=False):
    """out (+)= alpha * reduce(a over `axes`); out is contiguous with the kept
    axes of a in order (any shape with that many elements)."""
    shape = tuple(a.shape)
    nd = len(shape)
    axes = {ax % nd for ax in axes} if nd else set()
    mask = (L.C.c_int * max(1, nd))(*[1 if d in axes else 0 for d in range(nd)])
    shp = _i64(shape)
    ws_bytes = L.lib().mtx_reduce_workspace_bytes(nd, shp, mask)
    ws = dev.empty_buf((ws_bytes,), "uint8") if ws_bytes else None
    if not out.is_contiguous():
        raise ValueError("reduce output must be contiguous")
    L.call("mtx_reduce_f32", int(op), nd, shp, L.ptr(a), _i64(a.stride()), mask, L.ptr(out),
           float(alpha), int(bool(accumulate)), L.ptr(ws) if ws is not None else None, ws_bytes,
           L.stream_handle())
    return out


# ---------------------------------------------------------------------------
# GEMM
# ---------------------------------------------------------------------------

GEMM_ACT_NONE, GEMM_ACT_GELU, GEMM_ACT_GELU_BWD, GEMM_ACT_ADD = 0, 1, 2, 4


def gemm_ln_fits(M, K, N):
    """Whether mtx_gemm_ln_f32 takes an (M, K) @ (K, N) product."""
    return 1 <= M <= 64 and 1 <= K <= 4096 and 1 <= N <= 2048


def gemm_ln(a, b, c, gamma, beta_ln, eps, y, bias=None, alpha=1.0, beta=1.0):
    """c = alpha * a @ b + bias + beta * c, then y = LayerNorm(rows of c)
    with gamma, beta_ln, eps (mtx_gemm_ln_f32: a decode step's residual
    projection and the LayerNorm after it; a (M, K) with M <= 64, b (K, N),
    c and y (M, N) with unit column strides)."""
    M, K = a.shape[-2], a.shape[-1]
    N = b.shape[-1]
    for name, t in (("a", a), ("b", b), ("c", c), ("y", y), ("gamma", gamma), ("beta", beta_ln)):
        if _dt(t) != "float32":
            raise ValueError(f"gemm_ln: {name} must be fp32")
    if tuple(c.shape[-2:]) != (M, N) or tuple(y.shape[-2:]) != (M, N) or c.stride(-1) != 1 or y.stride(-1) != 1:
        raise ValueError(f"gemm_ln: c and y must be ({M}, {N}) with unit column strides")
    if gamma.numel() != N or beta_ln.numel() != N or not (gamma.is_contiguous() and beta_ln.is_contiguous()):
        raise ValueError(f"gemm_ln: gamma and beta must be contiguous with N={N} elements")
    ws_bytes = L.lib().mtx_gemm_ln_workspace_bytes(M, N, K)
    ws = dev.empty_buf((ws_bytes,), "uint8") if ws_bytes else None
    L.call("mtx_gemm_ln_f32", int(M), int(N), int(K), float(alpha), L.ptr(a), int(a.stride(-2)),
           int(a.stride(-1)), L.ptr(b), int(b.stride(-2)), int(b.stride(-1)), float(beta), L.ptr(c),
           int(c.stride(-2)), L.ptr(bias) if bias is not None else None, L.ptr(gamma), L.ptr(beta_ln),
           float(eps), L.ptr(y), int(y.stride(-2)), L.ptr(ws) if ws is not None else None, ws_bytes,
           L.stream_handle())
    return y


GEMM_FP32, GEMM_BF16X3 = L.MTX_GEMM_FP32, L.MTX_GEMM_BF16X3


def set_gemm_mode(mode: int) -> int:
    """Select how products of at least 128 x 128 are computed
    (mtx_gemm_set_mode): GEMM_BF16X3 (the default: fp32 values split into
    three bf16 pieces on the bf16 matrix cores, fp32-accurate) or GEMM_FP32
    (fp32 MFMA).  Returns the previous mode."""
    prev = int(L.lib().mtx_gemm_get_mode())
    L.call("mtx_gemm_set_mode", int(mode))
    return prev


def get_gemm_mode() -> int:
    return int(L.lib().mtx_gemm_get_mode())


def set_attn_mode(mode: int) -> int:
    """Select how fp32 attention with 64-wide heads computes its
    products (mtx_attn_set_mode): GEMM_BF16X3 (the default: three bf16
    pieces per fp32 value on the bf16 matrix cores) or GEMM_FP32 (fp32
    MFMA).  Returns the previous mode."""
    prev = int(L.lib().mtx_attn_get_mode())
    L.call("mtx_attn_set_mode", int(mode))
    return prev


def get_attn_mode() -> int:
    return int(L.lib().mtx_attn_get_mode())


ATTN_BWD_TWOPASS, ATTN_BWD_ONEPASS = L.ATTN_BWD_TWOPASS, L.ATTN_BWD_ONEPASS


def set_attn_bwd_mode(mode: int) -> int:
    """Select how the backward of bf16 attention with D <= 64 runs
    (mtx_attn_set_bwd_mode): ATTN_BWD_TWOPASS (the default: deterministic
    dQ and dK/dV passes) or ATTN_BWD_ONEPASS (one key-outer kernel writes
    dK/dV and adds dQ with fp32 atomics, after a delta kernel that zeroes
    dq).  Returns the previous mode."""
    prev = int(L.lib().mtx_attn_get_bwd_mode())
    L.call("mtx_attn_set_bwd_mode", int(mode))
    return prev


def get_attn_bwd_mode() -> int:
    return int(L.lib().mtx_attn_get_bwd_mode())


def attn_bwd_onepass_used(dtype: str, D: int) -> bool:
    """Whether attn_bwd (all phases, no dropout) takes the one-pass kernels
    for this input dtype and head size."""
    return dtype == "bfloat16" and D <= 64 and get_attn_bwd_mode() == ATTN_BWD_ONEPASS


@functools.lru_cache(maxsize=512)
def _gemm_workspace_bytes(M, N, K, batch):
    """mtx_gemm_workspace_bytes, a function of the sizes alone."""
    return L.lib().mtx_gemm_workspace_bytes(M, N, K, batch)


def gemm(a, b, c, alpha=1.0, beta=0.0, bias=None, M=None, N=None, K=None, batch=1,
         sa=None, sb=None, sc=None, act=GEMM_ACT_NONE, aux=None, colsum=None, colsum_accumulate=False):
    """C = alpha*A@B + beta*C (+bias) with explicit (row, col, batch) strides
    for each operand; defaults take them from 2-D/3-D tensors.  act/aux: the
    GELU epilogues of mtx_gemm_act_f32 (aux shaped like C: the pre-activation
    written by act 1, read by act 2), or GEMM_ACT_ADD: C = ... + aux (a
    residual stream, not C itself).  colsum: a contiguous (N,) tensor that
    receives (or, with colsum_accumulate, adds) the column sums of B -- a
    Linear layer's bias gradient next to its weight gradient
    (mtx_gemm_wgrad_f32: batch 1, alpha 1, no bias or activation)."""
    if sa is None:
        sa = (a.stride(-2), a.stride(-1), a.stride(0) if a.dim() == 3 else 0)
    if sb is None:
        sb = (b.stride(-2), b.stride(-1), b.stride(0) if b.dim() == 3 else 0)
    if sc is None:
        sc = (c.stride(-2), c.stride(-1), c.stride(0) if c.dim() == 3 else 0)
    M = a.shape[-2] if M is None else M
    K = a.shape[-1] if K is None else K
    N = b.shape[-1] if N is None else N
    for name, t in (("A", a), ("B", b), ("C", c), ("bias", bias), ("aux", aux)):
        if t is not None and _dt(t) != "float32":
            raise ValueError(f"gemm: {name} must be fp32 (got {t.dtype})")
    # one operand stride must be unit; otherwise the caller passes a copy
    ws_bytes = _gemm_workspace_bytes(int(M), int(N), int(K), int(batch))
    ws = dev.empty_buf((ws_bytes,), "uint8") if ws_bytes else None
    if colsum is not None:
        if batch != 1 or alpha != 1.0 or bias is not None or act != GEMM_ACT_NONE:
            raise ValueError("gemm: colsum needs batch 1, alpha 1 and no bias or activation")
        if _dt(colsum) != "float32" or colsum.numel() != N or not colsum.is_contiguous():
            raise ValueError(f"gemm: colsum must be a contiguous fp32 tensor of N={N} elements")
        L.call("mtx_gemm_wgrad_f32", int(M), int(N), int(K), L.ptr(a), int(sa[0]), int(sa[1]),
               L.ptr(b), int(sb[0]), int(sb[1]), float(beta), L.ptr(c), int(sc[0]), int(sc[1]),
               L.ptr(colsum), int(bool(colsum_accumulate)),
               L.ptr(ws) if ws is not None else None, ws_bytes, L.stream_handle())
        return c
    if act != GEMM_ACT_NONE:
        if aux is not None:
            if tuple(aux.shape[-2:]) != (M, N) or _dt(aux) != "float32":
                raise ValueError(f"gemm: aux must be fp32 with C's shape ({M}, {N})")
            sx = (aux.stride(-2), aux.stride(-1), aux.stride(0) if aux.dim() == 3 else 0)
        elif act in (GEMM_ACT_GELU_BWD, GEMM_ACT_ADD):
            raise ValueError("gemm: this epilogue needs aux")
        else:
            sx = (0, 0, 0)
        L.call("mtx_gemm_act_f32", int(M), int(N), int(K), int(batch),
               float(alpha), L.ptr(a), int(sa[0]), int(sa[1]), int(sa[2]),
               L.ptr(b), int(sb[0]), int(sb[1]), int(sb[2]),
               float(beta), L.ptr(c), int(sc[0]), int(sc[1]), int(sc[2]),
               L.ptr(bias) if bias is not None else None, int(act),
               L.ptr(aux) if aux is not None else None, int(sx[0]), int(sx[1]), int(sx[2]),
               L.ptr(ws) if ws is not None else None, ws_bytes, L.stream_handle())
        return c
    L.call("mtx_gemm_f32", int(M), int(N), int(K), int(batch),
           float(alpha), L.ptr(a), int(sa[0]), int(sa[1]), int(sa[2]),
           L.ptr(b), int(sb[0]), int(sb[1]), int(sb[2]),
           float(beta), L.ptr(c), int(sc[0]), int(sc[1]), int(sc[2]),
           L.ptr(bias) if bias is not None else None,
           L.ptr(ws) if ws is not None else None, ws_bytes, L.stream_handle())
    return c


# size limits of mtx_gemm_step_f32 (one-launch decode-step projections)
STEP_MAX_M, STEP_MAX_K = 64, 512
ACT_NONE, ACT_GELU = 0, 1


def step_fits(M, K):
    """True when mtx_gemm_step_f32 takes an (M, K) activation."""
    return 1 <= M <= STEP_MAX_M and 1 <= K <= STEP_MAX_K


def gemm_step(a, b, bias=None, c=None, beta=0.0, act=ACT_NONE, kv=None):
    """One decode-step projection: P = a @ b + bias, a (M, K) with unit k
    stride, b (K, N) with unit n stride.  Columns of P go to c (M, Nc) as
    act(P + beta*c); with kv = (kcache, vcache, lengths) the last 2*Ck columns
    go to the caches (B, T, Ck) at row lengths[m] - 1 instead (Nc = N - 2*Ck)."""
    M, Kd = a.shape
    N = b.shape[1]
    if a.stride(1) != 1 or b.stride(1) != 1 or b.shape[0] != Kd:
        raise ValueError("gemm_step: a (M, K) and b (K, N) need unit inner strides")
    if kv is not None:
        kc, vc, lengths = kv
        _need_cuda(kc, vc, lengths)
        Bc, T, Ck = kc.shape
        if tuple(vc.shape) != tuple(kc.shape) or tuple(vc.stride()) != tuple(kc.stride()) or kc.stride(2) != 1 \
                or Bc < M:
            raise ValueError("gemm_step: k/v caches must be (B >= M, T, C) with equal strides")
        if _dt(lengths) != "int32" or lengths.numel() < M:
            raise ValueError("gemm_step: lengths must be int32 with >= M entries")
        nc = N - 2 * Ck
        cache_args = (L.ptr(kc), L.ptr(vc), kc.stride(0), kc.stride(1), T, L.ptr(lengths))
    else:
        nc = N
        cache_args = (None, None, 0, 0, 0, None)
    if nc < 0:
        raise ValueError("gemm_step: N too small for the cache columns")
    if nc > 0:
        if c is None or tuple(c.shape) != (M, nc) or c.stride(1) != 1:
            raise ValueError(f"gemm_step: c must be ({M}, {nc}) with unit column stride")
    L.call("mtx_gemm_step_f32", int(M), int(N), int(Kd), L.ptr(a), a.stride(0), L.ptr(b), b.stride(0),
           float(beta), L.ptr(c) if nc > 0 else None, c.stride(0) if nc > 0 else 0,
           L.ptr(bias) if bias is not None else None, int(act), int(nc), *cache_args, L.stream_handle())
    return c


def greedy_pick(x, cur, ids, lengths, pos=None, margins=None, t_base=0):
    """mtx_greedy_pick_f32: per row of x (rows, cols) the first-maximum index
    to cur (int64 (rows,)) and to ids[lengths[row], row] (int64 (Tmax, rows)),
    the top-2 margin to margins[lengths[row] - t_base, row] (float32
    (n, rows)); then lengths += 1 (int32 (rows,)) and pos += 1."""
    _need_cuda(x, cur, ids, lengths)
    rows, cols = x.shape
    if _dt(x) != "float32" or x.stride(1) != 1:
        raise ValueError("greedy_pick: x must be fp32 with contiguous rows")
    if _dt(cur) != "int64" or cur.numel() != rows or not cur.is_contiguous():
        raise ValueError("greedy_pick: cur must be contiguous int64 (rows,)")
    if _dt(ids) != "int64" or ids.dim() != 2 or ids.shape[1] != rows or not ids.is_contiguous():
        raise ValueError("greedy_pick: ids must be contiguous int64 (Tmax, rows)")
    if _dt(lengths) != "int32" or lengths.numel() != rows or not lengths.is_contiguous():
        raise ValueError("greedy_pick: lengths must be contiguous int32 (rows,)")
    if pos is not None and _dt(pos) != "int64":
        raise ValueError("greedy_pick: pos must be int64")
    if margins is not None and (_dt(margins) != "float32" or margins.dim() != 2 or margins.shape[1] != rows
                                or not margins.is_contiguous()):
        raise ValueError("greedy_pick: margins must be contiguous fp32 (n, rows)")
    L.call("mtx_greedy_pick_f32", rows, cols, L.ptr(x), x.stride(0), L.ptr(cur), L.ptr(ids), ids.shape[0],
           L.ptr(margins) if margins is not None else None, int(t_base),
           margins.shape[0] if margins is not None else 0, L.ptr(lengths),
           L.ptr(pos) if pos is not None else None, L.stream_handle())


def embedding2_fwd(wa, ia, wb, ib, out, ib_stride=1):
    """out (n, C) = wa[ia] + wb[ib] (mtx_embedding2_fwd_f32); ib_stride 0
    broadcasts ib[0]."""
    Va, C = wa.shape
    Vb = wb.shape[0]
    n = ia.numel()
    if _dt(ia) != "int64" or _dt(ib) != "int64" or wb.shape[1] != C or out.shape[-1] != C:
        raise ValueError("embedding2: int64 ids and tables / output of one width")
    if wa.stride(1) != 1 or wb.stride(1) != 1 or out.stride(-1) != 1 or not ia.is_contiguous():
        raise ValueError("embedding2: rows must be contiguous")
    if ib_stride and ib.numel() < n:
        raise ValueError("embedding2: ib has fewer ids than ia")
    L.call("mtx_embedding2_fwd_f32", L.ptr(wa), wa.stride(0), Va, L.ptr(ia), L.ptr(wb), wb.stride(0), Vb,
           L.ptr(ib), int(ib_stride), L.ptr(out), out.stride(-2) if out.dim() >= 2 else C, n, C, L.stream_handle())
    return out


def embedding2_ln_fwd(wa, ia, wb, ib, out, gamma, beta, eps, y, ib_stride=1):
    """out (n, C) = wa[ia] + wb[ib] and y = LayerNorm(out) with gamma, beta,
    eps in one launch (mtx_embedding2_ln_fwd_f32)."""
    Va, C = wa.shape
    Vb = wb.shape[0]
    n = ia.numel()
    if _dt(ia) != "int64" or _dt(ib) != "int64" or wb.shape[1] != C or out.shape[-1] != C or y.shape[-1] != C:
        raise ValueError("embedding2_ln: int64 ids and tables / outputs of one width")
    if (wa.stride(1) != 1 or wb.stride(1) != 1 or out.stride(-1) != 1 or y.stride(-1) != 1
            or not ia.is_contiguous()):
        raise ValueError("embedding2_ln: rows must be contiguous")
    if gamma.numel() != C or beta.numel() != C or not (gamma.is_contiguous() and beta.is_contiguous()):
        raise ValueError("embedding2_ln: gamma and beta must be contiguous with C elements")
    if ib_stride and ib.numel() < n:
        raise ValueError("embedding2_ln: ib has fewer ids than ia")
    L.call("mtx_embedding2_ln_fwd_f32", L.ptr(wa), wa.stride(0), Va, L.ptr(ia), L.ptr(wb), wb.stride(0), Vb,
           L.ptr(ib), int(ib_stride), L.ptr(out), out.stride(-2) if out.dim() >= 2 else C, n, C,
           L.ptr(gamma), L.ptr(beta), float(eps), L.ptr(y), y.stride(-2) if y.dim() >= 2 else C,
           L.stream_handle())
    return y


def head_pick(x, w, bias, cur, ids, lengths, pos=None, margins=None, t_base=0, pending=None, ln=None):
    """mtx_head_pick_f32: logits = x @ w + bias per row of x (rows, K), w
    (K, V), then the pick of greedy_pick on them (cur, ids, margins,
    lengths, pos) in one launch.  With ln = (gamma, beta, eps) the rows are
    raw (plus pending = (ws, ks, bias) as in qkv_attn_step) and the product
    reads their LayerNorm."""
    _need_cuda(x, w, cur, ids, lengths)
    rows, Kd = x.shape
    V = w.shape[1]
    if _dt(x) != "float32" or _dt(w) != "float32" or x.stride(1) != 1 or w.stride(1) != 1:
        raise ValueError("head_pick: x and w must be fp32 with contiguous rows")
    if w.shape[0] != Kd or (bias is not None and (bias.numel() != V or not bias.is_contiguous())):
        raise ValueError("head_pick: w must be (K, V) and bias (V,)")
    if _dt(cur) != "int64" or cur.numel() != rows or not cur.is_contiguous():
        raise ValueError("head_pick: cur must be contiguous int64 (rows,)")
    if _dt(ids) != "int64" or ids.dim() != 2 or ids.shape[1] != rows or not ids.is_contiguous():
        raise ValueError("head_pick: ids must be contiguous int64 (Tmax, rows)")
    if _dt(lengths) != "int32" or lengths.numel() != rows or not lengths.is_contiguous():
        raise ValueError("head_pick: lengths must be contiguous int32 (rows,)")
    if pos is not None and _dt(pos) != "int64":
        raise ValueError("head_pick: pos must be int64")
    if margins is not None and (_dt(margins) != "float32" or margins.dim() != 2 or margins.shape[1] != rows
                                or not margins.is_contiguous()):
        raise ValueError("head_pick: margins must be contiguous fp32 (n, rows)")
    pargs, lnargs = _pending_args(pending, ln, rows, Kd)
    L.call("mtx_head_pick_f32", rows, Kd, V, L.ptr(x), x.stride(0), *pargs, *lnargs, L.ptr(w), w.stride(0),
           L.ptr(bias) if bias is not None else None, L.ptr(cur), L.ptr(ids), ids.shape[0],
           L.ptr(margins) if margins is not None else None, int(t_base),
           margins.shape[0] if margins is not None else 0, L.ptr(lengths),
           L.ptr(pos) if pos is not None else None, L.stream_handle())


# ---------------------------------------------------------------------------
# row kernels
# ---------------------------------------------------------------------------

def _rows(t):
    """(rows, L, leading stride) of a tensor whose last axis is contiguous and
    whose leading axes collapse to one row index."""
    if t.stride(-1) != 1:
        raise ValueError("last axis must be contiguous")
    Lx = t.shape[-1]
    rows = t.numel() // Lx if Lx else 0
    if t.dim() == 1:
        return 1, Lx, Lx
    # leading axes must collapse with a single stride
    ld = t.stride(-2)
    expect = ld * t.shape[-2]
    for d in range(t.dim() - 3, -1, -1):
        if t.shape[d] != 1 and t.stride(d) != expect:
            raise ValueError("leading axes do not collapse")
        expect *= t.shape[d]
    return rows, Lx, ld


def softmax_fwd(x, y, causal_tq=0, log=False):
    rx, Lx, ldx = _rows(x)
    _, _, ldy = _rows(y)
    L.call("mtx_softmax_fwd_f32", L.ptr(x), ldx, L.ptr(y), ldy, rx, Lx, int(causal_tq), int(log),
           L.stream_handle())
    return y


def softmax_bwd(y, dy, dx, log=False, accumulate=False):
    r, Lx, ldy = _rows(y)
    _, _, lddy = _rows(dy)
    _, _, lddx = _rows(dx)
    L.call("mtx_softmax_bwd_f32", L.ptr(y), ldy, L.ptr(dy), lddy, L.ptr(dx), lddx, r, Lx, int(log),
           int(bool(accumulate)), L.stream_handle())
    return dx


def layernorm_fwd(x, gamma, beta, y, mean, std, eps):
    r, C, ldx = _rows(x)
    _, _, ldy = _rows(y)
    L.call("mtx_layernorm_fwd_f32", L.ptr(x), ldx, L.ptr(gamma), L.ptr(beta), L.ptr(y), ldy,
           L.ptr(mean), L.ptr(std), r, C, float(eps), L.stream_handle())
    return y


def layernorm_bwd(x, gamma, mean, std, dy, dx=None, dgamma=None, dbeta=None, accumulate=False,
                  accumulate_params=None, addend=None):
    """dx and/or dgamma, dbeta in one pass over x and dy.  `accumulate` adds
    into dx; `accumulate_params` (default: same as `accumulate`) adds into
    dgamma and dbeta; `addend` (rows, C) is added to dx instead (dx = the
    LayerNorm gradient + addend; not with `accumulate`)."""
    if accumulate_params is None:
        accumulate_params = accumulate
    flags = (1 if accumulate else 0) | (2 if accumulate_params else 0)
    r, C, ldx = _rows(x)
    _, _, lddy = _rows(dy)
    lddx = _rows(dx)[2] if dx is not None else C
    ldadd = _rows(addend)[2] if addend is not None else 0
    ws = None
    ws_bytes = 0
    if dgamma is not None:
        ws_bytes = L.lib().mtx_layernorm_bwd_workspace_bytes(r, C)
        ws = dev.empty_buf((ws_bytes,), "uint8")
    L.call("mtx_layernorm_bwd_f32", L.ptr(x), ldx, L.ptr(gamma), L.ptr(mean), L.ptr(std),
           L.ptr(dy), lddy, L.ptr(dx) if dx is not None else None, lddx,
           L.ptr(addend) if addend is not None else None, ldadd,
           L.ptr(dgamma) if dgamma is not None else None, L.ptr(dbeta) if dbeta is not None else None,
           r, C, flags, L.ptr(ws) if ws is not None else None, ws_bytes,
           L.stream_handle())


def gelu_fwd(x, y):
    if not (x.is_contiguous() and y.is_contiguous()):
        raise ValueError("gelu: contiguous tensors only")
    L.call("mtx_gelu_fwd_f32", L.ptr(x), L.ptr(y), x.numel(), L.stream_handle())
    return y


def gelu_bwd(x, dy, dx, accumulate=False):
    if not (x.is_contiguous() and dy.is_contiguous() and dx.is_contiguous()):
        raise ValueError("gelu_bwd: contiguous tensors only")
    L.call("mtx_gelu_bwd_f32", L.ptr(x), L.ptr(dy), L.ptr(dx), x.numel(), int(bool(accumulate)),
           L.stream_handle())
    return dx


def xent_fwd(logits, labels, row_loss, lse):
    r, V, ld = _rows(logits)
    L.call("mtx_xent_fwd_f32", L.ptr(logits), ld, L.ptr(labels), L.ptr(row_loss), L.ptr(lse), r, V,
           L.stream_handle())


def xent_bwd(logits, labels, lse, gscalar, scale, dlogits, accumulate=False):
    r, V, ld = _rows(logits)
    _, _, ldd = _rows(dlogits)
    L.call("mtx_xent_bwd_f32", L.ptr(logits), ld, L.ptr(labels), L.ptr(lse), L.ptr(gscalar),
           float(scale), L.ptr(dlogits), ldd, r, V, int(bool(accumulate)), L.stream_handle())


TOP_MAX = 64  # alternatives per row of token_logprobs


def _logits_rows(logits, tokens, **vectors):
    """(dtype code, rows, V, ld) of the spec of (rows, V) logits, checked with
    those of the int64 (rows,) tokens and fp32 (rows,) vectors (None: not
    there) that go with them."""
    shape, strides, dtype = logits
    if len(shape) != 2 or strides[1] != 1:
        raise ValueError("logits must be (rows, V) with contiguous rows")
    rows, V = shape
    _vector("tokens", tokens, rows, "int64")
    for name, t in vectors.items():
        _vector(name, t, rows, "float32")
    return _code(_dt(dtype)), rows, V, strides[0]


@functools.lru_cache(maxsize=512)
def _logprobs_plan(logits, tokens, top, logprob, entropy, lse, top_ids, top_logprobs):
    code, rows, V, ld = _logits_rows(logits, tokens, logprob=logprob, entropy=entropy, lse=lse)
    if not 0 <= top <= min(V, TOP_MAX):
        raise ValueError(f"top must be between 0 and {min(V, TOP_MAX)} (got {top})")
    for name, t, dt in (("top_ids", top_ids, "int64"), ("top_logprobs", top_logprobs, "float32")):
        if _dt(t[2]) != dt or tuple(t[0]) != (rows, top) or (rows and top and not _packed(*t[:2])):
            raise ValueError(f"{name} must be contiguous {dt} ({rows}, {top})")
    dev.device()
    return code, rows, V, ld


def token_logprobs(logits, tokens, top: int = 0, scale: float = 1.0, logprob=None, entropy=None, lse=None,
                   top_ids=None, top_logprobs=None):
    """Log probabilities of one token per row of logits (rows, V), fp32 or
    bf16, at scale * logits (1e-27 to 1e38), the entropy, and the `top` (<= 64) most likely
    tokens with theirs, ties to the lowest id (mtx_token_logprobs).  A token
    outside [0, V) means the row has none (logprob 0).  Returns (logprob,
    entropy, lse) fp32 (rows,), top_ids int64 and top_logprobs fp32
    (rows, top)."""
    top, n = int(top), logits.shape[0]
    logprob, entropy, lse = (dev.empty_buf((n,), "float32") if t is None else t for t in (logprob, entropy, lse))
    if top_ids is None:
        top_ids = dev.empty_buf((n, max(0, top)), "int64")
    if top_logprobs is None:
        top_logprobs = dev.empty_buf((n, max(0, top)), "float32")
    if not (logits.is_cuda and tokens.is_cuda and logprob.is_cuda and entropy.is_cuda and lse.is_cuda
            and top_ids.is_cuda and top_logprobs.is_cuda):
        _on_device(logits, tokens, logprob, entropy, lse, top_ids, top_logprobs)
    code, rows, V, ld = _logprobs_plan(
        (logits.shape, logits.stride(), logits.dtype), (tokens.shape, tokens.stride(), tokens.dtype), top,
        (logprob.shape, logprob.stride(), logprob.dtype), (entropy.shape, entropy.stride(), entropy.dtype),
        (lse.shape, lse.stride(), lse.dtype), (top_ids.shape, top_ids.stride(), top_ids.dtype),
        (top_logprobs.shape, top_logprobs.stride(), top_logprobs.dtype))
    if dev.SEVERAL:
        _on_gpu0(logits, tokens, logprob, entropy, lse, top_ids, top_logprobs)
    if rows:
        L.call("mtx_token_logprobs", code, rows, V, logits.data_ptr(), ld, tokens.data_ptr(), float(scale),
               logprob.data_ptr(), lse.data_ptr(), entropy.data_ptr(), top, top_ids.data_ptr() if top else None,
               top_logprobs.data_ptr() if top else None, None, 0, L.stream_handle())
    return logprob, entropy, lse, top_ids, top_logprobs


@functools.lru_cache(maxsize=512)
def _logprobs_bwd_plan(logits, tokens, lse, entropy, g_logprob, g_entropy, dlogits):
    code, rows, V, ld = _logits_rows(logits, tokens, lse=lse, entropy=entropy, g_logprob=g_logprob,
                                     g_entropy=g_entropy)
    if _dt(dlogits[2]) != "float32" or tuple(dlogits[0]) != (rows, V) or dlogits[1][1] != 1:
        raise ValueError(f"dlogits must be fp32 ({rows}, {V}) with contiguous rows")
    dev.device()
    return code, rows, V, ld, dlogits[1][0]


def token_logprobs_bwd(logits, tokens, lse, entropy, g_logprob, g_entropy, scale: float = 1.0, dlogits=None,
                       accumulate: bool = False):
    """The logits' gradient from those of logprob and entropy (fp32 (rows,),
    None: 0) and the forward's lse and entropy (mtx_token_logprobs_bwd):
    fp32 (rows, V), added to dlogits with accumulate."""
    if dlogits is None:
        if accumulate:
            raise ValueError("accumulate needs dlogits")
        dlogits = dev.empty_buf(logits.shape, "float32")
    if not (logits.is_cuda and tokens.is_cuda and lse.is_cuda and entropy.is_cuda and dlogits.is_cuda):
        _on_device(logits, tokens, lse, entropy, dlogits)
    code, rows, V, ld, ldd = _logprobs_bwd_plan(
        (logits.shape, logits.stride(), logits.dtype), (tokens.shape, tokens.stride(), tokens.dtype),
        (lse.shape, lse.stride(), lse.dtype), (entropy.shape, entropy.stride(), entropy.dtype), _spec(g_logprob),
        _spec(g_entropy), (dlogits.shape, dlogits.stride(), dlogits.dtype))
    if dev.SEVERAL:
        _on_gpu0(logits, tokens, lse, entropy, g_logprob, g_entropy, dlogits)
    if rows:
        L.call("mtx_token_logprobs_bwd", code, rows, V, logits.data_ptr(), ld, tokens.data_ptr(), lse.data_ptr(),
               entropy.data_ptr(), _ptr(g_logprob), _ptr(g_entropy), float(scale), dlogits.data_ptr(), ldd,
               1 if accumulate else 0, L.stream_handle())
    return dlogits


def embedding_fwd(weight, idx, out):
    V, C = weight.shape
    L.call("mtx_embedding_fwd_f32", L.ptr(weight), weight.stride(0), V, L.ptr(idx), idx.numel(),
           L.ptr(out), C, C, L.stream_handle())
    return out


def embedding_bwd(idx, grad, dweight, accumulate=False):
    """dweight (+)= scatter-add of grad rows by idx.  Small tables use a
    one-hot GEMM on MFMA (onehot^T @ grad); large ones the row-owner kernel.
    Both are deterministic."""
    V, C = dweight.shape
    n = idx.numel()
    if V <= 4096 and n * V <= (1 << 27):
        onehot = dev.empty_buf((n, V), "float32")
        L.call("mtx_onehot_f32", L.ptr(idx), n, V, L.ptr(onehot), L.stream_handle())
        gemm(onehot.t(), grad, dweight, beta=1.0 if accumulate else 0.0, M=V, N=C, K=n, batch=1,
             sa=(1, V, 0), sb=(grad.stride(0), grad.stride(1), 0), sc=(dweight.stride(0), dweight.stride(1), 0))
        return dweight
    L.call("mtx_embedding_bwd_f32", L.ptr(idx), idx.numel(), L.ptr(grad), C, L.ptr(dweight),
           dweight.stride(0), V, C, int(bool(accumulate)), L.stream_handle())
    return dweight


# ---------------------------------------------------------------------------
# training with a large vocabulary
# ---------------------------------------------------------------------------

def _matrix(name, spec, shape=None):
    """(shape, row stride, dtype) of a (rows, cols) view with contiguous rows."""
    got, strides, dtype = spec
    if len(got) != 2 or (shape is not None and tuple(got) != shape):
        want = "(rows, cols)" if shape is None else shape
        raise ValueError(f"{name} must be {want}, got shape {tuple(got)}")
    rows, cols = got
    if strides[1] != 1 and cols != 1:
        raise ValueError(f"{name} must have contiguous rows")
    ld = strides[0] if rows > 1 else cols
    if ld < cols:
        raise ValueError(f"{name}: its rows overlap")
    return (rows, cols), ld, _dt(dtype)


def _int32(**sizes):
    """Sizes that the library takes as 32-bit numbers, to which a call would wrap them."""
    for name, size in sizes.items():
        if size >= 1 << 31:
            raise ValueError(f"{name} must be below 2^31 (got {size})")


@functools.lru_cache(maxsize=512)
def _lookup_plan(weight, ids, out):
    (V, C), ldw, dtype = _matrix("weight", weight)
    n = ids[0][0] if len(ids[0]) == 1 else -1
    _vector("ids", ids, n, "int64")
    _, ldo, odt = _matrix("out", out, (n, C))
    if not V or not C:
        raise ValueError(f"weight of shape {(V, C)} has no rows")
    _int32(C=C)
    dev.device()
    return (_code(dtype), _code(odt)), (ldw, V), (n, C), ldo


def embedding_lookup(weight, ids, scale: float = 1.0, out=None):
    """out[i] = scale * weight[ids[i]] for a (V, C) table, fp32 or bf16, and int64
    (n,) ids (mtx_embedding_lookup); zeros for an id outside [0, V): padding.
    out: (n, C), fp32 or bf16 (default: like the table)."""
    if out is None:
        out = dev.empty_buf((ids.shape[0], weight.shape[1]), _dt(weight))
    if not (weight.is_cuda and ids.is_cuda and out.is_cuda):
        _on_device(weight, ids, out)
    codes, table, (n, C), ldo = _lookup_plan((weight.shape, weight.stride(), weight.dtype),
                                             (ids.shape, ids.stride(), ids.dtype), (out.shape, out.stride(), out.dtype))
    if dev.SEVERAL:
        _on_gpu0(weight, ids, out)
    if n:
        L.call("mtx_embedding_lookup", *codes, weight.data_ptr(), *table, ids.data_ptr(), n, C, float(scale),
               out.data_ptr(), ldo, L.stream_handle())
    return out


@functools.lru_cache(maxsize=512)
def _grad_plan(ids, grad, dweight):
    (V, C), lddw, wdt = _matrix("dweight", dweight)
    if wdt != "float32":
        raise ValueError("dweight must be fp32")
    if not V or not C:
        raise ValueError(f"dweight of shape {(V, C)} has no rows")
    _int32(C=C)
    n = ids[0][0] if len(ids[0]) == 1 else -1
    _vector("ids", ids, n, "int64")
    _, ldg, dtype = _matrix("grad", grad, (n, C))
    dev.device()
    return _code(dtype), n, ldg, (lddw, V, C), L.lib().mtx_embedding_grad_workspace_bytes(_code(dtype), n, V, C)


def embedding_grad(ids, grad, dweight, scale: float = 1.0, accumulate: bool = False):
    """dweight (V, C) fp32 = (with accumulate: +=) scale * the rows of grad (n, C),
    fp32 or bf16, added up by their int64 (n,) ids in a fixed order
    (mtx_embedding_grad).  Rows whose id is outside [0, V) add to nothing."""
    if not (ids.is_cuda and grad.is_cuda and dweight.is_cuda):
        _on_device(ids, grad, dweight)
    code, n, ldg, table, ws_bytes = _grad_plan((ids.shape, ids.stride(), ids.dtype),
                                               (grad.shape, grad.stride(), grad.dtype),
                                               (dweight.shape, dweight.stride(), dweight.dtype))
    if dev.SEVERAL:
        _on_gpu0(ids, grad, dweight)
    ws = dev.empty_buf((ws_bytes,), "uint8") if ws_bytes else None
    L.call("mtx_embedding_grad", code, ids.data_ptr() if n else None, n, grad.data_ptr() if n else None, ldg,
           float(scale), dweight.data_ptr(), *table, 1 if accumulate else 0, _ptr(ws), ws_bytes, L.stream_handle())
    return dweight


@functools.lru_cache(maxsize=512)
def _dropout_plan(x, residual, out):
    (rows, cols), ldx, dtype = _matrix("x", x)
    lds = [ldx]
    for name, spec in (("residual", residual), ("out", out)):
        if spec is None:
            lds.append(cols)
            continue
        _, ld, dt = _matrix(name, spec, (rows, cols))
        if dt != dtype:
            raise ValueError(f"{name} must be {dtype} like x (got {dt})")
        lds.append(ld)
    dev.device()
    return _code(dtype), rows, cols, lds


def dropout(x, p: float, seed: int, offset: int = 0, residual=None, out=None, subsequence: int = 0, base=None):
    """(residual +) x * keep / (1 - p) over a (rows, cols) view, fp32 or bf16, the
    keep-mask drawn where it is used (mtx_dropout): dropout_keep_philox's at
    (seed, offset), with the generator's `subsequence`; p = 0 keeps everything.  The
    gradient is the same call on the upstream gradient; out may be x or residual.  base:
    a device int64 (1,) array that is added to offset when the kernel runs.  Returns
    out."""
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout probability must be in [0, 1) (got {p})")
    if out is None:
        out = dev.empty_buf(x.shape, _dt(x))
    if not (x.is_cuda and out.is_cuda):
        _on_device(x, out)
    if residual is not None:
        _on_device(residual)
    code, rows, cols, (ldx, ldr, ldo) = _dropout_plan((x.shape, x.stride(), x.dtype), _spec(residual),
                                                      (out.shape, out.stride(), out.dtype))
    if base is not None:
        _on_device(base)
        _vector("base", _spec(base), 1, "int64")
    if dev.SEVERAL:
        _on_gpu0(*(t for t in (x, residual, out, base) if t is not None))
    if rows and cols:
        L.call("mtx_dropout", code, x.data_ptr(), ldx, _ptr(residual), ldr, out.data_ptr(), ldo, rows, cols, p,
               1.0 / (1.0 - p), int(seed) & (2**64 - 1), int(offset) & (2**64 - 1), int(subsequence) & (2**32 - 1),
               _ptr(base), L.stream_handle())
    return out


def _either_order(name, spec, shape):
    """(row stride, column stride, dtype) of a matrix that is contiguous along
    its rows or its columns."""
    got, strides, dtype = spec
    if len(got) != 2 or (shape is not None and tuple(got) != shape):
        raise ValueError(f"{name} must be {'(C, V)' if shape is None else shape}, got shape {tuple(got)}")
    (rows, cols), (sr, sc) = got, strides
    # strides of an axis of one element mean nothing
    if cols == 1:
        sc = 1 if sr != 1 or rows == 1 else rows
    if rows == 1 and sc == 1:
        sr = cols
    if not ((sc == 1 and sr >= cols) or (sr == 1 and sc >= rows)):
        raise ValueError(f"{name}: its rows or its columns must be contiguous and not overlap (strides "
                         f"{tuple(strides)})")
    return sr, sc, _dt(dtype)


@functools.lru_cache(maxsize=512)
def _xent_plan(x, w, labels, bias, loss, row_loss, lse, dx, dw, db, logits_bytes, one_piece):
    (n, C), ldx, dtype = _matrix("x", x)
    code = _code(dtype)
    swc, swv, wdt = _either_order("w", w, None)
    V = w[0][1]
    if w[0][0] != C or wdt != dtype or not C or not V:
        raise ValueError(f"w must be ({C}, V) {dtype} like x, got {tuple(w[0])} {wdt}")
    _int32(C=C, V=V)
    _vector("labels", labels, n, "int64")
    for name, t, size in (("bias", bias, V), ("loss", loss, 1), ("row_loss", row_loss, n), ("lse", lse, n),
                          ("db", db, V)):
        _vector(name, t, size, "float32")
    if db is not None and bias is None:
        raise ValueError("db without a bias")
    gdt, lddx, sdc, sdv = None, C, V, 1
    if dx is not None:
        _, lddx, gdt = _matrix("dx", dx, (n, C))
    if dw is not None:
        sdc, sdv, other = _either_order("dw", dw, (C, V))
        if gdt not in (None, other):
            raise ValueError(f"dx and dw must share a dtype (got {gdt}, {other})")
        gdt = other
    if gdt is None and db is not None:
        gdt = "float32"
    if gdt is not None and gdt not in ("float32", dtype):
        raise ValueError(f"gradients of {dtype} inputs must be float32 or {dtype} (got {gdt})")
    if one_piece and gdt != "bfloat16":
        raise ValueError(f"one_piece is for bfloat16 gradients (got {gdt})")
    dev.device()
    gcode = -1 if gdt is None else _code(gdt) | (L.MTX_GRAD_ONE_PIECE if one_piece else 0)
    ws = L.lib().mtx_linear_xent_workspace_bytes(code, gcode, n, C, V, 0 if db is None else 1, logits_bytes)
    return (code, gcode, n, C, V), ldx, (swc, swv), lddx, (sdc, sdv), ws


def linear_xent(x, w, labels, bias=None, loss=None, row_loss=None, lse=None, dx=None, dw=None, db=None,
                logits_bytes: int = 1 << 31, one_piece: bool = False):
    """Softmax cross-entropy of the logits x @ w + bias, and its gradients, a block of
    rows' logits at a time (mtx_linear_xent).  x (n, C) and w (C, V), contiguous along
    either axis (a (V, C) table's .t()), fp32 or bf16; labels int64 (n,), one outside
    [0, V): none (with dw, x must be finite there too); bias fp32 (V,).  Returns (loss
    (1,): the mean over the rows that have a label, row_loss (n,), lse (n,)), fp32.
    dx (n, C), dw (C, V) and db (V,), where given, receive the gradients of loss: fp32,
    dx and dw also bf16 with bf16 inputs.  bf16 gradients are off by the rounding of the result; with one_piece the
    logits' gradient is rounded to bf16 too (small vocabularies: not), for less time
    (8192 x 1024, V = 50021: 3.1 ms in place of 5.1, an error of 1.86e-3 of the norm in
    place of 1.66e-3).  A block's logits fill at most
    logits_bytes; beside them bf16 inputs take as much again for bf16 gradients, half
    of it more for fp32 ones.  No output may overlap an input or another output."""
    if logits_bytes < 1:
        raise ValueError(f"logits_bytes must be positive (got {logits_bytes})")
    n = x.shape[0]
    loss = dev.empty_buf((1,), "float32") if loss is None else loss
    row_loss, lse = (dev.empty_buf((n,), "float32") if t is None else t for t in (row_loss, lse))
    if not (x.is_cuda and w.is_cuda and labels.is_cuda and loss.is_cuda and row_loss.is_cuda and lse.is_cuda):
        _on_device(x, w, labels, loss, row_loss, lse)
    _on_device(*(t for t in (bias, dx, dw, db) if t is not None))
    sizes, ldx, sw, lddx, sd, ws_bytes = _xent_plan(
        (x.shape, x.stride(), x.dtype), (w.shape, w.stride(), w.dtype), (labels.shape, labels.stride(), labels.dtype),
        _spec(bias), (loss.shape, loss.stride(), loss.dtype), (row_loss.shape, row_loss.stride(), row_loss.dtype),
        (lse.shape, lse.stride(), lse.dtype), _spec(dx), _spec(dw), _spec(db), int(logits_bytes), bool(one_piece))
    if dev.SEVERAL:
        _on_gpu0(*(t for t in (x, w, labels, bias, loss, row_loss, lse, dx, dw, db) if t is not None))
    ws = dev.empty_buf((ws_bytes,), "uint8")
    L.call("mtx_linear_xent", *sizes, x.data_ptr(), ldx, w.data_ptr(), *sw, _ptr(bias), labels.data_ptr(),
           loss.data_ptr(), row_loss.data_ptr(), lse.data_ptr(), _ptr(dx), lddx, _ptr(dw), *sd, _ptr(db), int(logits_bytes),
           ws.data_ptr(), ws_bytes, L.stream_handle())
    return loss, row_loss, lse


class AdamTable:
    """Device table for the one-launch multi-tensor Adam (layout of the C
    struct AdamEntry: p, g, m, v, n, block0 -- six 64-bit words)."""

    def __init__(self, params, grads, ms, vs):
        n = len(params)
        sizes = (L.C.c_int64 * n)(*[p.numel() for p in params])
        b0 = (L.C.c_int64 * n)()
        total = L.C.c_int64()
        L.call("mtx_adam_blocks", sizes, n, b0, L.C.byref(total))
        rows = []
        for i in range(n):
            rows.append([params[i].data_ptr(), grads[i].data_ptr(), ms[i].data_ptr(), vs[i].data_ptr(),
                         params[i].numel(), b0[i]])
        host = np.array(rows, dtype=np.int64).reshape(n, 6)
        self.table = dev.from_host(host, np.int64).t
        self.n = n
        self.total_blocks = int(total.value)


def adam_bias_table(beta1, beta2, first_step, length):
    """Host float32 table of the bias corrections (1 - beta1^t, 1 - beta2^t)
    for steps first_step .. first_step + length - 1, entry (t - 1) % length."""
    out = np.empty(2 * length, dtype=np.float32)
    L.call("mtx_adam_bias_table", float(beta1), float(beta2), int(first_step), int(length),
           out.ctypes.data_as(L.C.c_void_p))
    return out


def adam_step_dev(table: AdamTable, lr, beta1, beta2, eps, weight_decay, step_dev, bias_dev):
    """Adam with the step count in device memory (step_dev int32 (1,),
    incremented by the launch) and bias corrections from bias_dev (2*len
    float32, adam_bias_table): a launch that replays unchanged in a graph."""
    L.call("mtx_adam_dev_f32", L.ptr(table.table), table.n, table.total_blocks, float(lr), float(beta1),
           float(beta2), float(eps), float(weight_decay), L.ptr(step_dev), L.ptr(bias_dev),
           bias_dev.numel() // 2, L.stream_handle())


def zero_grads(table: AdamTable):
    """Zero every gradient the table points at, in one launch."""
    L.call("mtx_zero_grads_f32", L.ptr(table.table), table.n, table.total_blocks, L.stream_handle())


def adam_step(table: AdamTable, lr, beta1, beta2, eps, weight_decay, step):
    L.call("mtx_adam_f32", L.ptr(table.table), table.n, table.total_blocks, float(lr), float(beta1),
           float(beta2), float(eps), float(weight_decay), int(step), L.stream_handle())
