"""The operators of training with a large vocabulary, as cases that can be timed
and checked one by one.

A case is a dict of plain sizes; ``prepare`` makes what a program has in hand
before the call, ``run`` is one pass through an operator, in plain torch or,
where ``own`` is true, through the package's entry points, and ``exact`` the
same numbers from the definition in 64 bits.  Operators (``op``):

  lookup   rows of an embedding table, scaled; a token outside the table has
           none and gets zeros (kernels.embedding_lookup)
  grad     the table's gradient: the tokens' rows added up by token
           (kernels.embedding_grad)
  dropout  inverted dropout, optionally added to a residual stream, whose mask
           comes from a counter-based generator and is never stored
           (kernels.dropout; the gradient is the same call on the gradient)
  xent     a vocabulary projection with its softmax cross entropy, and the
           gradients, without keeping the logits (kernels.linear_xent)
"""
import math

import torch

own = False

# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # a training batch of the 384-wide character model
        dict(name="lookup_chars", op="lookup", n=16384, V=65, C=384, dtype="float32", out="float32", scale=1.0,
             none=0.0),
        # a subword table in bf16, scaled by the square root of its width, contexts padded
        dict(name="lookup_words", op="lookup", n=32768, V=50021, C=1024, dtype="bfloat16", out="bfloat16", scale=32.0,
             none=0.1),
        # the character table's gradient: every token has hundreds of rows
        dict(name="grad_chars", op="grad", n=16384, V=65, C=384, dtype="float32", scale=1.0, none=0.0),
        # a few sentences of a subword vocabulary: most of the table gets nothing
        dict(name="grad_few", op="grad", n=300, V=5003, C=384, dtype="float32", scale=1.0, none=0.0),
        # a batch of the subword model: few frequent tokens, many rare ones
        dict(name="grad_words", op="grad", n=32768, V=50021, C=1024, dtype="bfloat16", scale=32.0, none=0.1),
        # a block's dropout and residual, the 384-wide model's training batch
        dict(name="drop_block", op="dropout", rows=16384, cols=384, p=0.1, dtype="float32", residual=True),
        # one context of the small character model: latency
        dict(name="drop_small", op="dropout", rows=32, cols=64, p=0.25, dtype="float32", residual=False),
        # a wide model's gradient in bf16
        dict(name="drop_wide", op="dropout", rows=32768, cols=2048, p=0.1, dtype="bfloat16", residual=False),
        # the character vocabulary's head and loss over a training batch
        dict(name="head_chars", op="xent", n=16384, C=384, V=65, dtype="float32", grads="float32", tied=False, bias=True,
             none=0.0),
        # the same with a subword vocabulary of odd size
        dict(name="head_words", op="xent", n=8192, C=384, V=5003, dtype="float32", grads="float32", tied=False, bias=True,
             none=0.0),
        # a bf16 model whose head is its embedding table, contexts padded: the largest
        dict(name="head_tied", op="xent", n=8192, C=1024, V=50021, dtype="bfloat16", grads="bfloat16", tied=True,
             bias=False, none=0.1),
        # scoring a few hundred tokens: no gradients
        dict(name="head_score", op="xent", n=500, C=1024, V=50021, dtype="bfloat16", grads="", tied=False, bias=True,
             none=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST_ROWS = 2 * 32768 * 1024  # values of the largest batch of embedded tokens
_MOST_TABLE = 50021 * 1024  # and of the largest table
_MOST_LOGITS = 8192 * 50021


def draw(rng):
    op = rng.choice(["lookup", "grad", "grad", "dropout", "xent", "xent"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "dropout":
        cols = rng.choice([_log(rng, 1, 8192), 64 * rng.randint(1, 64)])
        most = 32768 * 2048 // (2 if dtype == "float32" else 1)
        return dict(op=op, rows=max(1, min(_log(rng, 1, 65536), most // cols)), cols=cols,
                    p=rng.choice([0.1, 0.1, 0.25, 0.5, 0.9]), dtype=dtype, residual=rng.random() < 0.5)
    if op in ("lookup", "grad"):
        C = rng.choice([_log(rng, 1, 4096), 64 * rng.randint(1, 32)])
        V = max(1, min(_log(rng, 2, 131072), _MOST_TABLE // C))
        n = max(1, min(_log(rng, 1, 131072), _MOST_ROWS // (2 * C)))
        case = dict(op=op, n=n, V=V, C=C, dtype=dtype, scale=rng.choice([1.0, round(math.sqrt(C), 3)]),
                    none=rng.choice([0.0, 0.0, 0.3]))
        return dict(case, out=rng.choice(["float32", dtype])) if op == "lookup" else case
    C = rng.choice([_log(rng, 8, 2048), 64 * rng.randint(1, 32)])
    V = max(2, min(_log(rng, 2, 131072), _MOST_TABLE // C))
    n = max(1, min(_log(rng, 1, 16384), _MOST_LOGITS // V, 8192 * 50021 * 1024 // (V * C)))
    if dtype == "float32":  # as much time as the largest in bf16
        n = max(1, n // 2)
    grads = rng.choice(["", dtype, dtype, "float32"])
    return dict(op=op, n=n, C=C, V=V, dtype=dtype, grads=grads, tied=rng.random() < 0.5, bias=rng.random() < 0.5,
                none=rng.choice([0.0, 0.0, 0.3]))


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6007 + 17)
    return g


def _normal(g, shape, std, dtype):
    return torch.randn(tuple(shape), generator=g, device="cuda", dtype=dtype).mul_(std)


def _tokens(g, n, V, none):
    """n token ids whose frequencies fall as words' do (a token's is one over its
    rank), a share `none` of them -1: padding."""
    rank = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(V + 1)).long() - 1
    ids = torch.randperm(V, generator=g, device="cuda")[rank.clamp(0, V - 1)]
    pad = torch.rand(n, generator=g, device="cuda") < none
    return torch.where(pad, torch.full_like(ids, -1), ids)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    dt = getattr(torch, case["dtype"])
    f = dict(dtype=torch.float32, device="cuda")
    if op == "dropout":
        shape = (case["rows"], case["cols"])
        st = dict(op=op, x=_normal(g, shape, 1.0, dt), p=case["p"], out=torch.empty(shape, dtype=dt, device="cuda"))
        st["residual"] = _normal(g, shape, 1.0, dt) if case["residual"] else None
        # where the generator stands: anywhere, also past 32 bits
        st["seed"] = int(seed) * 2654435761 % (1 << 63)
        st["offset"] = (int(seed) * 40503 << 16) % (1 << 40)
        return st
    if op in ("lookup", "grad"):
        n, V, C = case["n"], case["V"], case["C"]
        st = dict(op=op, ids=_tokens(g, n, V, case["none"]), scale=case["scale"])
        if op == "lookup":
            st["weight"] = _normal(g, (V, C), 0.02, dt)
            st["out"] = torch.empty((n, C), dtype=getattr(torch, case["out"]), device="cuda")
        else:
            st["grad"] = _normal(g, (n, C), 1e-3, dt)
            st["dweight"] = torch.empty((V, C), **f)
        return st
    n, C, V = case["n"], case["C"], case["V"]
    labels = _tokens(g, n, V, case["none"])
    # logits of deviation 2.5, and rows that know something of their label
    table = _normal(g, (V, C), 2.5 / math.sqrt(C), dt)
    x = _normal(g, (n, C), 1.0, torch.float32)
    x += 2 * torch.rand((n, 1), generator=g, device="cuda") * table[labels.clamp(min=0)].float()
    st = dict(op=op, x=x.to(dt), labels=labels, w=table.t() if case["tied"] else table.t().contiguous(),
              bias=_normal(g, (V,), 0.5, torch.float32) if case["bias"] else None)
    del table
    st.update(loss=torch.empty(1, **f), row_loss=torch.empty(n, **f), lse=torch.empty(n, **f))
    if case["grads"]:
        out = dict(dtype=getattr(torch, case["grads"]), device="cuda")
        st["dx"] = torch.empty((n, C), **out)
        st["dw"] = torch.empty((V, C), **out).t() if case["tied"] else torch.empty((C, V), **out)
        st["db"] = torch.empty(V, **f) if case["bias"] else None
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(st):
    if own:
        return _OWN[st["op"]](st)
    return _PLAIN[st["op"]](st)


def _own_lookup(st):
    from minitorch_amd import kernels as K

    return K.embedding_lookup(st["weight"], st["ids"], scale=st["scale"], out=st["out"])


def _own_grad(st):
    from minitorch_amd import kernels as K

    return K.embedding_grad(st["ids"], st["grad"], st["dweight"], scale=st["scale"])


def _own_dropout(st):
    from minitorch_amd import kernels as K

    return K.dropout(st["x"], st["p"], st["seed"], st["offset"], residual=st["residual"], out=st["out"])


def _own_xent(st):
    from minitorch_amd import kernels as K

    out = [st["loss"], st["row_loss"], st["lse"]]
    if "dx" not in st:
        K.linear_xent(st["x"], st["w"], st["labels"], bias=st["bias"], loss=out[0], row_loss=out[1], lse=out[2])
        return out
    K.linear_xent(st["x"], st["w"], st["labels"], bias=st["bias"], loss=out[0], row_loss=out[1], lse=out[2],
                  dx=st["dx"], dw=st["dw"], db=st["db"])
    return out + [st["dx"], st["dw"]] + ([] if st["db"] is None else [st["db"]])


def _plain_lookup(st):
    ids, w = st["ids"], st["weight"]
    some = (ids >= 0) & (ids < w.shape[0])
    rows = w[torch.where(some, ids, torch.zeros_like(ids))].float() * st["scale"]
    return torch.where(some[:, None], rows, torch.zeros_like(rows)).to(st["out"].dtype)


def _plain_grad(st):
    ids, g, V = st["ids"], st["grad"].float(), st["dweight"].shape[0]
    # the rows without a token are added to one behind the table
    at = torch.where((ids >= 0) & (ids < V), ids, torch.full_like(ids, V))
    total = torch.zeros((V + 1, g.shape[1]), dtype=torch.float32, device="cuda").index_add_(0, at, g)
    return total[:V] * st["scale"]


_LOW = 0xFFFFFFFF


def _uniform(n, seed, offset):
    """n numbers in [0, 1) of 24 bits: words of Philox4x32-10 (Salmon, Moraes, Dror
    and Shaw, SC'11) with key `seed` and counters from `offset` on, in 64-bit
    integers whose low halves hold the words."""
    ctr = torch.arange((n + 3) // 4, dtype=torch.int64, device="cuda") + offset
    c0, c1 = ctr & _LOW, (ctr >> 32) & _LOW
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    for r in range(10):
        k0, k1 = (seed + r * 0x9E3779B9) & _LOW, ((seed >> 32) + r * 0xBB67AE85) & _LOW
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64
        c0, c1, c2, c3 = ((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW
    words = torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]
    return (words >> 8).float() * 2.0 ** -24


def _plain_dropout(st):
    x, p = st["x"], torch.tensor(st["p"], dtype=torch.float32, device="cuda")
    keep = _uniform(x.numel(), st["seed"], st["offset"]).reshape(x.shape) > p
    y = torch.where(keep, x.float() * float(1.0 / (1.0 - st["p"])), torch.zeros((), device="cuda"))
    if st["residual"] is not None:
        y = st["residual"].float() + y
    return y.to(x.dtype)


def _plain_xent(st):
    x, w, labels = st["x"].float(), st["w"].float(), st["labels"]
    V = w.shape[1]
    some = (labels >= 0) & (labels < V)
    at = torch.where(some, labels, torch.zeros_like(labels))[:, None]
    z = x @ w
    if st["bias"] is not None:
        z += st["bias"]
    m = z.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(-1, keepdim=True))
    row_loss = torch.where(some, (lse - z.gather(1, at))[:, 0], torch.zeros((), device="cuda"))
    count = some.sum().clamp(min=1)
    out = [(row_loss.sum() / count).reshape(1), row_loss, lse[:, 0]]
    if "dx" not in st:
        return out
    z -= lse
    d = z.exp_()
    d.scatter_add_(1, at, torch.full_like(d[:, :1], -1.0))
    d *= (some / count)[:, None]
    out += [(d @ w.t()).to(st["dx"].dtype), (x.t() @ d).to(st["dw"].dtype)]
    return out + ([] if st["db"] is None else [d.sum(0)])


_OWN = dict(lookup=_own_lookup, grad=_own_grad, dropout=_own_dropout, xent=_own_xent)
_PLAIN = dict(lookup=_plain_lookup, grad=_plain_grad, dropout=_plain_dropout, xent=_plain_xent)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------
_SIZE = {"": 0, "float32": 4, "bfloat16": 2}


def work(case):
    op, size = case["op"], _SIZE[case["dtype"]]
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return dict(bytes=n * size * (3 if case["residual"] else 2), flops=2 * n)
    if op in ("lookup", "grad"):
        n, V, C = case["n"], case["V"], case["C"]
        rows = int(n * (1 - case["none"]))
        if op == "lookup":  # a row that several tokens ask for is read once
            return dict(bytes=min(rows, V) * C * size + n * (C * _SIZE[case["out"]] + 8), flops=n * C)
        return dict(bytes=rows * C * size + 8 * n + 4 * V * C, flops=rows * C)
    n, C, V, out = case["n"], case["C"], case["V"], _SIZE[case["grads"]]
    more = 4 * V * (2 if out else 1) if case["bias"] else 0
    return dict(bytes=(n + V) * C * (size + out) + 16 * n + more, flops=(6 if out else 2) * n * V * C)


def exact(case, seed):
    st = prepare(case, seed)
    return _EXACT[case["op"]](case, st)


def _exact_lookup(case, st):
    table = torch.nn.functional.pad(st["weight"].double(), (0, 0, 0, 1))  # a row of zeros for no token
    return table[st["ids"]] * st["scale"]


def _exact_grad(case, st):
    V, C = st["dweight"].shape
    total = torch.zeros((V + 1, C), dtype=torch.float64, device="cuda")
    total.index_put_((st["ids"],), st["grad"].double(), accumulate=True)
    return total[:V] * st["scale"]


def _exact_dropout(case, st):
    import numpy as np

    n = case["rows"] * case["cols"]
    if n > 1 << 24:
        return None
    # the generator in numpy's unsigned integers, word for word as it is defined
    low, half = np.uint64(_LOW), np.uint64(32)
    at = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(st["offset"])
    c = [at & low, at >> half, np.zeros_like(at), np.zeros_like(at)]
    key = [np.uint64(st["seed"]) & low, np.uint64(st["seed"]) >> half]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> half) ^ c[1] ^ key[0], b & low, (a >> half) ^ c[3] ^ key[1], a & low]
        key = [(key[0] + np.uint64(0x9E3779B9)) & low, (key[1] + np.uint64(0xBB67AE85)) & low]
    u = (np.stack(c, 1).reshape(-1)[:n] >> np.uint64(8)).astype(np.float64) / 2 ** 24
    keep = torch.from_numpy(u > np.float64(np.float32(st["p"]))).cuda().reshape(st["x"].shape)
    y = st["x"].double() * keep / (1.0 - st["p"])
    return y if st["residual"] is None else st["residual"].double() + y


def _exact_xent(case, st):
    x, w, labels = st["x"].double(), st["w"].double(), st["labels"]
    z = torch.mm(x, w)
    if st["bias"] is not None:
        z += st["bias"].double()
    logp = torch.log_softmax(z, -1)
    lse = z[:, 0] - logp[:, 0]
    del z
    has = (labels >= 0).nonzero()[:, 0]
    row_loss = torch.zeros(len(labels), dtype=torch.float64, device="cuda")
    row_loss[has] = -logp[has, labels[has]]
    out = [row_loss.sum().reshape(1) / max(1, len(has)), row_loss, lse]
    if not case["grads"]:
        return out
    d = logp.exp_()
    d[has, labels[has]] -= 1
    d[labels < 0] = 0
    d /= max(1, len(has))
    out += [torch.mm(d, w.t()), torch.mm(x.t(), d)]
    return out + [d.sum(0)] if case["bias"] else out


_EXACT = dict(lookup=_exact_lookup, grad=_exact_grad, dropout=_exact_dropout, xent=_exact_xent)
