"""The operators of serving from a paged key-value cache and of log
probabilities, as cases that can be timed and checked one by one.

A case is a dict of plain sizes; ``prepare`` makes what a program has in hand
before the call, ``run`` is one pass through an operator, in plain torch or,
where ``own`` is true, through the package's entry points, and ``exact`` the
same numbers from the definition in 64 bits.  Operators (``op``):

  append   keys and values of new tokens written into a cache's pages
           (kernels.kv_append_paged)
  decode   attention of one new token per sequence over its pages, with grouped
           heads, and the weight each cached row received
           (kernels.attn_decode_paged)
  evict    a cache cut down to the rows that received the most weight and the
           latest ones (kernels.kv_evict_paged)
  logprobs log probabilities of given tokens, the entropy and the top
           alternatives, and the gradient of the first two
           (kernels.token_logprobs, kernels.token_logprobs_bwd)

Pages are (pages, K/V heads, rows, head size) views; a page table holds each
sequence's pages in order, -1 where it has none.
"""
import math

import torch

own = False

# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one decode step of the six-head character model, a few sequences
        dict(name="decode_chars", op="decode", B=8, H=6, Hkv=6, D=64, L=200, low=20, page=16, q="float32",
             cache="float32", layout="rows", weights=False, idle=0),
        # a full batch of that model with its cache in bf16, pages of an odd size
        dict(name="decode_mixed", op="decode", B=64, H=6, Hkv=6, D=64, L=1000, low=1, page=20, q="float32",
             cache="bfloat16", layout="heads", weights=False, idle=0),
        # one long document: few rows, a long axis
        dict(name="decode_one_long", op="decode", B=1, H=8, Hkv=1, D=128, L=131071, low=131071, page=32,
             q="bfloat16", cache="bfloat16", layout="heads", weights=False, idle=0),
        # a serving batch of long contexts with grouped heads, the largest
        dict(name="decode_batch_long", op="decode", B=16, H=32, Hkv=8, D=128, L=16384, low=8000, page=64,
             q="bfloat16", cache="bfloat16", layout="heads", weights=False, idle=0),
        # a step whose attention weights are accumulated for eviction, ragged
        # lengths and slots of the batch that hold no sequence
        dict(name="decode_weights", op="decode", B=32, H=16, Hkv=4, D=64, L=4099, low=60, page=16, q="bfloat16",
             cache="bfloat16", layout="rows", weights=True, idle=2),
        # a step's new rows: fp32 rows into a bf16 cache
        dict(name="append_step", op="append", B=64, T=1, Hkv=6, D=64, page=16, rows="float32", cache="bfloat16",
             layout="rows", past=250),
        # a batch of ragged prompts
        dict(name="append_prompt", op="append", B=16, T=2000, Hkv=8, D=128, page=64, rows="bfloat16",
             cache="bfloat16", layout="heads", past=0),
        # the character model's caches cut back to three quarters
        dict(name="evict_chars", op="evict", B=32, Hkv=6, D=64, L=256, low=200, keep=192, recent=32, page=16,
             cache="float32", layout="rows"),
        # long contexts cut down to a budget
        dict(name="evict_long", op="evict", B=8, Hkv=8, D=128, L=40000, low=30000, keep=8192, recent=512, page=64,
             cache="bfloat16", layout="heads"),
        # one step's answers: few rows of a subword vocabulary with alternatives
        dict(name="logprobs_step", op="logprobs", rows=8, V=50021, top=20, dtype="bfloat16", scale=1.25, train=False),
        # scoring the character model's contexts
        dict(name="logprobs_chars", op="logprobs", rows=16384, V=65, top=5, dtype="float32", scale=1.0, train=False),
        # training on log probabilities with an entropy term
        dict(name="logprobs_train", op="logprobs", rows=4096, V=50021, top=0, dtype="float32", scale=1.0, train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST = 16 * 12192 * 8 * 128  # values of K in the largest decode case


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "append", "evict", "logprobs", "logprobs"])
    if op == "logprobs":
        V = _log(rng, 2, 131072)
        rows = _log(rng, 1, max(1, min(16384, 4096 * 50021 // V)))
        train = rng.random() < 0.5
        # whole rows are sorted by the plain form: its alternatives come from fewer rows
        top = 0 if train and rng.random() < 0.7 else min(V, rng.randint(1, 32))
        if top:
            rows = min(rows, max(1, (1 << 24) // V))
        return dict(op=op, rows=rows, V=V, top=top, dtype=rng.choice(["float32", "bfloat16"]),
                    scale=rng.choice([1.0, 1.25, 0.7]), train=train)
    D = rng.choice([16, 32, 64, 64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 6, 8])
    page = rng.choice([1, 8, 16, 16, 20, 32, 64, 128, 37])
    kinds = [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("bfloat16", "bfloat16")]
    rows, cache = rng.choice(kinds)
    layout = rng.choice(["heads", "rows"])
    B = _log(rng, 1, 96)
    most = _MOST // (2 if cache == "float32" else 1)
    if op == "append":
        T = _log(rng, 1, 4096)
        B = max(1, min(B, most // 4 // (T * Hkv * D)))
        return dict(op=op, B=B, T=T, Hkv=Hkv, D=D, page=page, rows=rows, cache=cache, layout=layout,
                    past=rng.choice([0, rng.randint(1, 300)]))
    L = _log(rng, 1, 65536)
    B = max(1, min(B, most // (L * Hkv * D)))
    L = min(L, most // (B * Hkv * D))
    low = rng.randint(1, L)
    if op == "evict":
        keep = rng.randint(1, L)
        return dict(op=op, B=B, Hkv=Hkv, D=D, L=L, low=low, keep=keep, recent=rng.randint(0, keep), page=page,
                    cache=cache, layout=layout)
    return dict(op=op, B=B, H=Hkv * rng.choice([1, 1, 2, 3, 4, 8, 8, 20]), Hkv=Hkv, D=D, L=L, low=low, page=page,
                q=rows, cache=cache, layout=layout, weights=rng.random() < 0.4, idle=rng.choice([0, 0, 1]))


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _normal(g, shape, std, dtype):
    return torch.randn(tuple(shape), generator=g, device="cuda", dtype=dtype).mul_(std)


def _spread(low, high, n):
    """n whole numbers spread evenly from high down to low: a batch's lengths."""
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """Cached rows of each sequence (all of them, in a fixed order)."""
    if case["op"] == "append":
        return [case["past"] + n for n in _counts(case)]
    n = _spread(case["low"], case["L"], case["B"])
    for i in range(min(case.get("idle", 0), case["B"] - 1)):
        n[-1 - i] = 0
    return n


def _counts(case):
    return _spread((case["T"] + 1) // 2, case["T"], case["B"])


def _table(g, lengths, page, spare=0):
    """A page table over shuffled pages, and how many pages there are."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(need))
    col = torch.arange(width, device="cuda")
    n = torch.tensor(need, device="cuda")
    at = (torch.cumsum(n, 0) - n)[:, None] + col
    held = col < n[:, None]
    return torch.where(held, ids[at.clamp(max=max(0, total - 1))], torch.full_like(at, -1, dtype=torch.int32)), ids, total


def _pages(g, n, case, dtype):
    """A (pages, heads, rows, size) view of a pool stored by heads or by rows."""
    h, p, d = case["Hkv"], case["page"], case["D"]
    if case["layout"] == "heads":
        return _normal(g, (n, h, p, d), 1.0, dtype)
    return _normal(g, (n, p, h, d), 1.0, dtype).transpose(1, 2)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "logprobs":
        rows, V = case["rows"], case["V"]
        logits = _normal(g, (rows, V), 2.5, getattr(torch, case["dtype"]))
        # mostly tokens the model finds likely, as sampled ones are
        tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
        likely = logits.argmax(-1)
        tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.3, likely, tokens)
        f = dict(dtype=torch.float32, device="cuda")
        st = dict(op=op, logits=logits, tokens=tokens, top=case["top"], scale=case["scale"],
                  logprob=torch.empty(rows, **f), entropy=torch.empty(rows, **f), lse=torch.empty(rows, **f),
                  top_ids=torch.empty((rows, case["top"]), dtype=torch.int64, device="cuda"),
                  top_logprobs=torch.empty((rows, case["top"]), **f))
        if case["train"]:
            st.update(g_logprob=_normal(g, (rows,), 1.0 / rows, torch.float32),
                      g_entropy=_normal(g, (rows,), 0.1 / rows, torch.float32),
                      dlogits=torch.empty((rows, V), **f))
        return st
    cache = getattr(torch, case["cache"])
    lengths = _lengths(case)
    st = dict(op=op, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if op == "evict":
        width = -(-case["keep"] // case["page"])
        more = case["B"] * width
        st["table"], ids, total = _table(g, lengths, case["page"], more)
        st["to"] = ids[total - more:].view(case["B"], width).contiguous()
        st["keep"], st["recent"] = case["keep"], case["recent"]
        cap = st["table"].shape[1] * case["page"]
        shape = (case["B"], case["Hkv"], cap)
        # weights that accumulated over steps: a few rows hold most of them;
        # rows that no step looked at have none
        w = torch.exp(_normal(g, shape, 2.0, torch.float32))
        w[torch.rand(shape, generator=g, device="cuda") < 0.15] = 0.0
        st["weights"] = w
        st["weights_to"] = torch.empty_like(w)
        st["slots"] = torch.empty((case["B"], case["Hkv"], case["keep"]), dtype=torch.int32, device="cuda")
        st["lengths_to"] = torch.empty_like(st["lengths"])
    else:
        st["table"], _, total = _table(g, lengths, case["page"])
        cap = st["table"].shape[1] * case["page"]
    st["k_pages"], st["v_pages"] = (_pages(g, max(1, total), case, cache) for _ in range(2))
    if op == "append":
        dt = getattr(torch, case["rows"])
        B, T, h, d = case["B"], case["T"], case["Hkv"], case["D"]
        # (B, T, heads, size) as a projection leaves them, read by heads
        st["k"], st["v"] = (_normal(g, (B, T, h, d), 1.0, dt).transpose(1, 2) for _ in range(2))
        st["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
    elif op == "decode":
        dt = getattr(torch, case["q"])
        B, H, D = case["B"], case["H"], case["D"]
        st["q"] = _normal(g, (B, H, 1, D), 2.0, dt)  # scores of deviation 2
        st["scale"] = 1.0 / math.sqrt(D)
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty((B, H), dtype=torch.float32, device="cuda")
        if case["weights"]:
            shape = (B, case["Hkv"], cap)
            st["weights"] = torch.rand(shape, generator=g, device="cuda")
            st["weights_to"] = torch.zeros(shape, device="cuda")
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(st):
    if own:
        return _OWN[st["op"]](st)
    return _PLAIN[st["op"]](st)


def _own_append(st):
    from minitorch_amd import kernels as K

    K.kv_append_paged(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], counts=st["counts"])
    return [st["k_pages"], st["v_pages"]]


def _own_decode(st):
    from minitorch_amd import kernels as K

    if "weights" not in st:
        K.attn_decode_paged(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["scale"],
                            out=st["out"], lse=st["lse"])
        return [st["out"], st["lse"]]
    K.attn_decode_paged(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["scale"],
                        out=st["out"], lse=st["lse"], weights=st["weights_to"], weights_in=st["weights"])
    return [st["out"], st["lse"], st["weights_to"]]


def _own_evict(st):
    from minitorch_amd import kernels as K

    K.kv_evict_paged(st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["weights"], st["to"], st["keep"],
                     st["recent"], lengths_out=st["lengths_to"], weights_out=st["weights_to"], slots=st["slots"])
    return [st["k_pages"], st["v_pages"], st["lengths_to"], st["weights_to"], st["slots"]]


def _own_logprobs(st):
    from minitorch_amd import kernels as K

    K.token_logprobs(st["logits"], st["tokens"], top=st["top"], scale=st["scale"], logprob=st["logprob"],
                     entropy=st["entropy"], lse=st["lse"], top_ids=st["top_ids"], top_logprobs=st["top_logprobs"])
    out = [st["logprob"], st["entropy"], st["lse"], st["top_ids"], st["top_logprobs"]]
    if "dlogits" in st:
        K.token_logprobs_bwd(st["logits"], st["tokens"], st["lse"], st["entropy"], st["g_logprob"], st["g_entropy"],
                             scale=st["scale"], dlogits=st["dlogits"])
        out.append(st["dlogits"])
    return out


def _places(table, rows, n_pages, page):
    """Page and place of each row of `rows` (B, ...), and whether it has one."""
    flat = table.gather(1, (rows // page).clamp(min=0, max=table.shape[1] - 1).reshape(rows.shape[0], -1))
    at = flat.reshape(rows.shape).long()
    held = (rows >= 0) & (rows < table.shape[1] * page) & (at >= 0) & (at < n_pages)
    return torch.where(held, at, torch.zeros_like(at)), rows.clamp(min=0) % page, held


def _plain_append(st):
    k, v, kp, vp = st["k"], st["v"], st["k_pages"], st["v_pages"]
    i = torch.arange(k.shape[2], device="cuda")
    n = st["counts"].long()[:, None]
    rows = torch.where(i < n, st["lengths"].long()[:, None] - n + i, torch.full_like(i, -1))
    at, place, held = _places(st["table"], rows, kp.shape[0], kp.shape[2])
    b, t = held.nonzero(as_tuple=True)
    kp[at[b, t], :, place[b, t]] = k[b, :, t].to(kp.dtype)
    vp[at[b, t], :, place[b, t]] = v[b, :, t].to(vp.dtype)
    return [kp, vp]


def _plain_decode(st):
    q, kp, vp, table = st["q"], st["k_pages"], st["v_pages"], st["table"]
    (B, H, _, D), h, page = q.shape, kp.shape[1], kp.shape[2]
    j = torch.arange(table.shape[1] * page, device="cuda").expand(B, -1)
    at, place, held = _places(table, j, kp.shape[0], page)
    held &= j < st["lengths"][:, None]
    at = torch.where(held, at, torch.zeros_like(at))
    k = kp[at, :, place].float().transpose(1, 2)  # (B, heads, rows, D)
    s = (q.float().reshape(B, h, H // h, D) @ k.transpose(-1, -2)) * st["scale"]
    seen = held[:, None, None]
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    v = vp[at, :, place].float().transpose(1, 2).masked_fill(~held[:, None, :, None], 0.0)
    some = torch.where(total == 0, torch.ones_like(total), total)
    out = [((p @ v) / some).reshape(B, H, 1, D).to(q.dtype), (m + torch.log(total)).reshape(B, H)]
    if "weights" in st:
        w = st["weights"] + (p / some).sum(2)
        out.append(torch.where((j < st["lengths"][:, None])[:, None], w, st["weights_to"]))
    return out


def _plain_evict(st):
    kp, vp, w, n = st["k_pages"], st["v_pages"], st["weights"], st["lengths"].long()
    keep, recent, page = st["keep"], st["recent"], kp.shape[2]
    B, h, cap = w.shape
    j = torch.arange(cap, device="cuda")
    n3 = n[:, None, None]
    rank = torch.where(j >= n3, torch.full_like(w, -math.inf), torch.where(j >= n3 - recent, torch.full_like(w, math.inf), w))
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    new = n.clamp(max=keep)
    i = torch.arange(first.shape[-1], device="cuda")
    none = torch.full_like(first, cap)
    slots = torch.sort(torch.where(i < new[:, None, None], first, none), dim=-1).values
    slots = torch.where(slots < cap, slots, torch.full_like(slots, -1))
    slots = torch.nn.functional.pad(slots, (0, keep - slots.shape[-1]), value=-1)
    kept = torch.gather(w, 2, slots.clamp(min=0))
    kept = torch.where(slots >= 0, kept, torch.zeros_like(kept))
    w_to = torch.zeros_like(w)
    w_to[..., :min(keep, cap)] = kept[..., :cap]
    at, place, held = _places(st["table"], slots, kp.shape[0], page)
    rows = torch.arange(keep, device="cuda").expand(B, -1)
    to_at, to_place, to_held = _places(st["to"], rows, kp.shape[0], page)
    b, hh, r = (held & to_held[:, None]).nonzero(as_tuple=True)
    to, frm = (to_at[b, r], hh, to_place[b, r]), (at[b, hh, r], hh, place[b, hh, r])
    kp[to] = kp[frm]
    vp[to] = vp[frm]
    return [kp, vp, new.to(torch.int32), w_to, slots.to(torch.int32)]


def _plain_logprobs(st):
    logits, tok, scale, top = st["logits"], st["tokens"], st["scale"], st["top"]
    x = logits.float() * scale
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    x -= lse  # log probabilities
    p = torch.exp(x)
    entropy = -(p * x).sum(-1)
    at = tok[:, None]
    out = [x.gather(1, at)[:, 0], entropy, lse[:, 0]]
    if top:
        ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top]
        out += [ids, x.gather(1, ids)]
    else:
        out += [st["top_ids"], st["top_logprobs"]]
    if "dlogits" in st:
        g, gh = st["g_logprob"][:, None], st["g_entropy"][:, None]
        d = p * (-g - gh * (x + entropy[:, None]))
        d.scatter_add_(1, at, g)
        out.append(d * scale)
    return out


_OWN = dict(append=_own_append, decode=_own_decode, evict=_own_evict, logprobs=_own_logprobs)
_PLAIN = dict(append=_plain_append, decode=_plain_decode, evict=_plain_evict, logprobs=_plain_logprobs)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------
_SIZE = {"float32": 4, "bfloat16": 2}


def work(case):
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["V"]
        size = _SIZE[case["dtype"]]
        per_row = 20 + 12 * case["top"]
        if not case["train"]:
            return dict(bytes=n * size + case["rows"] * per_row, flops=6 * n)
        return dict(bytes=n * (size + 4) + case["rows"] * (per_row + 8), flops=12 * n)
    lengths = _lengths(case)
    row = case["Hkv"] * case["D"] * _SIZE[case["cache"]]
    pages = sum(-(-n // case["page"]) for n in lengths)
    if op == "append":
        n = sum(_counts(case))
        return dict(bytes=2 * n * (row + case["Hkv"] * case["D"] * _SIZE[case["rows"]]) + 4 * pages, flops=0)
    n = sum(lengths)
    if op == "evict":
        kept = sum(min(x, case["keep"]) for x in lengths)
        cap = max(1, max(-(-x // case["page"]) for x in lengths)) * case["page"]
        return dict(bytes=4 * kept * row + 4 * case["Hkv"] * (n + case["B"] * (cap + case["keep"])) + 4 * pages,
                    flops=n * case["Hkv"])
    q = case["B"] * case["H"]
    more = 8 * n * case["Hkv"] if case["weights"] else 0
    return dict(bytes=2 * n * row + 2 * q * case["D"] * _SIZE[case["q"]] + 4 * q + 4 * pages + more,
                flops=4 * n * case["H"] * case["D"] + 4 * n * case["H"])


def exact(case, seed):
    """append and evict only move values: nothing there is computed."""
    if case["op"] == "decode":
        return _exact_decode(prepare(case, seed), _lengths(case))
    if case["op"] == "logprobs":
        return _exact_logprobs(prepare(case, seed))
    return None


def _exact_decode(st, lengths):
    kp, vp = st["k_pages"], st["v_pages"]
    q = st["q"].double()[:, :, 0]
    B, H, D = q.shape
    h, page = kp.shape[1], kp.shape[2]
    o, lse = torch.zeros_like(q), torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    w = st["weights_to"].double() if "weights" in st else None
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        ids = st["table"][b, :-(-n // page)].long()
        for i in range(h):
            k = kp[ids, i].double().reshape(-1, D)[:n]
            v = vp[ids, i].double().reshape(-1, D)[:n]
            part = slice(i * (H // h), (i + 1) * (H // h))
            logp = torch.log_softmax(torch.mm(q[b, part], k.t().contiguous()) * st["scale"], -1)
            s0 = torch.mm(q[b, part], k[:1].t().contiguous())[:, 0] * st["scale"]
            lse[b, part] = s0 - logp[:, 0]
            p = logp.exp()
            o[b, part] = torch.mm(p, v)
            if w is not None:
                w[b, i, :n] = st["weights"][b, i, :n].double() + p.sum(0)
    out = [o[:, :, None], lse]
    return out + [w] if w is not None else out


def _exact_logprobs(st):
    logits, tok = st["logits"], st["tokens"]
    rows, V = logits.shape
    parts = [[] for _ in range(6)]
    train = "dlogits" in st
    for r in range(0, rows, 512):
        part = slice(r, r + 512)
        logp = torch.log_softmax(logits[part].double() * st["scale"], -1)
        p = logp.exp()
        entropy = -torch.special.xlogy(p, p).sum(-1)
        lse = logits[part, 0].double() * st["scale"] - logp[:, 0]
        parts[0].append(logp.gather(1, tok[part, None])[:, 0])
        parts[1].append(entropy)
        parts[2].append(lse)
        if st["top"]:
            parts[4].append(torch.topk(logp, st["top"], dim=-1).values)
        if train:
            hot = torch.nn.functional.one_hot(tok[part], V)
            g, gh = st["g_logprob"][part, None].double(), st["g_entropy"][part, None].double()
            parts[5].append(((hot - p) * g - gh * p * (logp + entropy[:, None])) * st["scale"])
    out = [torch.cat(x) for x in parts[:3]]
    out += [None, torch.cat(parts[4]) if st["top"] else None]
    return out + [torch.cat(parts[5])] if train else out
