"""The steps of a decoding loop around its paged cache, as cases that can be timed and compared.

Three operators, beside the projections, rotary positions and attention of a layer:

* ``plan``: what a step's requests need of the cache: pages taken from and given back to a ring of
  free ones, page tables, starts, lengths, positions and slots (``cache_plan_forward``);
* ``prefix``: attention of each sequence's new tokens over a prefix that all sequences share and
  over its own pages (``prefix_cache_attention_forward``);
* ``sample``: a token per row of logits by temperature, top-k, top-p and min-p from a given random
  number (``sample_forward``).

A case is a dict of plain values.  ``listed()`` names twelve, ``draw(rng)`` gives more of the same
ranges.  ``prepare`` makes what a program holds before the call, ``run`` makes the call: elementary
torch operations where ``own`` is false, the library's operators where it is true.  ``exact``
restates the operator in 64 bits.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TORCH_DTYPE = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
               "int32": torch.int32, "int64": torch.int64}
ELEM_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # A small decoding batch between two steps: latency.
        {"name": "plan_tokens", "op": "plan", "b": 8, "n_lo": 1, "n_hi": 1, "len_lo": 17, "len_hi": 1025, "ended": 0,
         "page": 16, "pad": 0},
        # A large decoding batch in a captured step: some requests end, rows are padded.
        {"name": "plan_batch", "op": "plan", "b": 512, "n_lo": 1, "n_hi": 1, "len_lo": 130, "len_hi": 8192, "ended": 19,
         "page": 16, "pad": 64},
        # Prompts coming in beside decoding requests: many pages at once.
        {"name": "plan_prompts", "op": "plan", "b": 96, "n_lo": 1, "n_hi": 8192, "len_lo": 1, "len_hi": 4000, "ended": 11,
         "page": 16, "pad": 0},
        # Four conversations behind a system prompt: latency.
        {"name": "prefix_few", "op": "prefix", "b": 4, "n_lo": 1, "n_hi": 1, "prefix": 2000, "len_lo": 33, "len_hi": 300,
         "hq": 32, "hkv": 8, "d": 128, "page": 16, "dtype": "bfloat16"},
        # A decoding batch behind a long one: what such a service spends its time on.
        {"name": "prefix_tokens", "op": "prefix", "b": 64, "n_lo": 1, "n_hi": 1, "prefix": 8192, "len_lo": 20,
         "len_hi": 1100, "hq": 32, "hkv": 8, "d": 128, "page": 16, "dtype": "bfloat16"},
        # New questions and decoding requests together, groups of three heads, pages of 32, odd lengths.
        {"name": "prefix_mixed", "op": "prefix", "b": 12, "n_lo": 1, "n_hi": 300, "prefix": 2501, "len_lo": 301,
         "len_hi": 800, "hq": 24, "hkv": 8, "d": 64, "page": 32, "dtype": "float16"},
        # A float32 model's candidates of one text.
        {"name": "prefix_f32", "op": "prefix", "b": 16, "n_lo": 1, "n_hi": 1, "prefix": 4097, "len_lo": 1, "len_hi": 129,
         "hq": 12, "hkv": 12, "d": 64, "page": 16, "dtype": "float32"},
        # Sixteen questions to one long document: bound by the matrix cores.
        {"name": "prefix_questions", "op": "prefix", "b": 16, "n_lo": 128, "n_hi": 128, "prefix": 16384, "len_lo": 128,
         "len_hi": 128, "hq": 32, "hkv": 8, "d": 128, "page": 16, "dtype": "bfloat16"},
        # One conversation's next token: latency.
        {"name": "sample_one", "op": "sample", "b": 1, "v": 32000, "filter": "top_k_p", "dtype": "float16"},
        # A decoding batch over a large vocabulary by top-p.
        {"name": "sample_top_p", "op": "sample", "b": 64, "v": 131072, "filter": "top_p", "dtype": "bfloat16"},
        # Requests with settings of their own, greedy ones among them, an odd vocabulary.
        {"name": "sample_mixed", "op": "sample", "b": 33, "v": 50021, "filter": "mixed", "dtype": "float32"},
        # Many continuations by temperature alone: bound by reading the logits.
        {"name": "sample_many", "op": "sample", "b": 256, "v": 131072, "filter": "none", "dtype": "float32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "prefix", "prefix", "sample", "sample"])
    if op == "plan":
        hi = 1 if rng.random() < 0.5 else _log(rng, 2, 8192)
        case = {"op": op, "b": _log(rng, 1, 2000), "n_lo": 1, "n_hi": hi, "len_lo": rng.randint(0, 200),
                "len_hi": _log(rng, 200, 16384), "ended": rng.choice([0, 0, 5, 13]),
                "page": rng.choice([16, 16, 32, 64, 24, 1]), "pad": rng.choice([0, 0, 3, 500])}
        while case["b"] > 1 and (sum(n for n, _ in _requests(case)) > 1 << 16 or
                                 case["b"] * (case["len_hi"] + hi) > (1 << 22) * case["page"]):
            case["b"] = (case["b"] + 1) // 2
        return case
    if op == "sample":
        case = {"op": op, "b": _log(rng, 1, 512), "v": _log(rng, 500, 262144),
                "filter": rng.choice(["none", "top_k", "top_p", "top_k_p", "min_p", "mixed"]),
                "dtype": rng.choice(["float32", "float16", "bfloat16", "bfloat16"])}
        while case["b"] * case["v"] > 1 << 25:
            case["b"] = (case["b"] + 1) // 2
        return case
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    hkv = rng.choice([1, 2, 4, 5, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8]) if hkv <= 8 else 1
    hi = _log(rng, 1, 2048)
    n_hi = 1 if rng.random() < 0.6 else _log(rng, 1, hi)
    case = {"op": op, "b": _log(rng, 1, 96), "n_lo": 1 if rng.random() < 0.6 else n_hi, "n_hi": n_hi,
            "prefix": _log(rng, 16, 16384), "len_lo": rng.randint(max(1, n_hi), hi), "len_hi": hi, "hq": hkv * group,
            "hkv": hkv, "d": rng.choice([64, 64, 128, 128, 128, 40, 80, 96, 256]), "page": rng.choice([16, 16, 32, 64, 24]),
            "dtype": dtype}
    most = 4e11 if dtype != "float32" else 4e10              # operations of a pass
    while case["b"] > 1 and (work(case)["flops"] > most or
                             case["b"] * case["hq"] * case["n_hi"] * (case["prefix"] + case["len_hi"]) > 1 << 31):
        case["b"] = (case["b"] + 1) // 2
    while work(case)["flops"] > most:
        case["n_hi"] = (case["n_hi"] + 1) // 2
        case["n_lo"] = min(case["n_lo"], case["n_hi"])
    return case


# ------------------------------------------------------------------------ sizes ---
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _chunks(b, lo, hi):
    """New tokens of each of b requests: the most in the middle, single ones around it."""
    return [max(lo, int(round(hi ** (1 - abs(2 * i - b + 1) / max(b, 2))))) if hi > lo else hi for i in range(b)]


def _sequences(case):
    """(new tokens, length) of each sequence."""
    lens = _spread(case["len_lo"], case["len_hi"], case["b"])
    return [(min(n, l), l) for n, l in zip(_chunks(case["b"], case["n_lo"], case["n_hi"]), lens)]


def _requests(case):
    """(new tokens, tokens in the cache) of each request; -1 new tokens: it has ended."""
    past = _spread(case["len_lo"], case["len_hi"], case["b"])
    news = _chunks(case["b"], case["n_lo"], case["n_hi"])
    return [(-1 if case["ended"] and i % case["ended"] == case["ended"] // 2 else n, p)
            for i, (n, p) in enumerate(zip(news, past))]


def _pages_of(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["op"] == "plan":
        page, rows, moved = case["page"], case["pad"], 0
        for n, p in _requests(case):
            rows += max(n, 0)
            moved += _pages_of(p, page) if n < 0 else _pages_of(p + n, page) - _pages_of(p, page)
        return {"bytes": 4 * (4 * case["b"] + 1 + 2 * rows + 2 * moved) + 48, "flops": 0}
    e = ELEM_BYTES[case["dtype"]]
    if case["op"] == "sample":
        return {"bytes": case["b"] * (case["v"] * e + 28), "flops": 8 * case["b"] * case["v"]}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    seqs = _sequences(case)
    tokens = sum(n for n, _ in seqs)
    pairs = tokens * case["prefix"] + sum(n * (l - n) + n * (n + 1) // 2 for n, l in seqs)
    return {"bytes": e * d * (2 * tokens * hq + 2 * (case["prefix"] + sum(l for _, l in seqs)) * hkv),
            "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------- inputs ---
FILTERS = {"none": (0, 1.0, 0.0), "top_k": (1, 1.0, 0.0), "top_p": (0, 0.0, 0.0), "top_k_p": (1, 0.0, 0.0),
           "min_p": (0, 1.0, 1.0)}


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    host = torch.Generator()
    host.manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(TORCH_DTYPE[case["dtype"]])

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=DEVICE)

    def shuffled(v):
        return [v[i] for i in torch.randperm(len(v), generator=host).tolist()]

    if case["op"] == "plan":
        req, page = shuffled(_requests(case)), case["page"]
        have = torch.tensor([_pages_of(p, page) for _, p in req])
        need = torch.tensor([_pages_of(p + max(n, 0), page) for n, p in req])
        cols, used = int(need.max()) + 1, int(have.sum())
        total = used + int((need - have).sum()) + 64
        order = torch.randperm(total, generator=host).to(torch.int32)
        # the first pages of the order lie in the tables' rows, the others in the ring of free ones
        table = torch.zeros(len(req), cols, dtype=torch.int32)
        owned = torch.arange(cols) < have[:, None]
        table[owned] = order[:used]
        taken = int(torch.randint(0, 5 * total, (1,), generator=host))
        free = torch.full((total,), -1, dtype=torch.int32)
        free[(taken + torch.arange(total - used)) % total] = order[used:]
        rows = sum(max(n, 0) for n, _ in req) + case["pad"]
        return {"new": ints([n for n, _ in req]), "past": ints([p for _, p in req]), "pages": table.to(DEVICE),
                "free": free.to(DEVICE), "state": ints([taken, taken + total - used, 0], torch.int64),
                "offset": ints([int(torch.randint(0, 4000, (1,), generator=host))]), "rows": rows}
    if case["op"] == "sample":
        b, v = case["b"], case["v"]
        # a bulk of tokens that hardly matter and a few in each row that stand out
        x = torch.randn(b, v, generator=g, device=DEVICE) * 2.0
        x += 10.0 * (1.0 - torch.rand(b, v, generator=g, device=DEVICE) * (v / 12)).clamp(min=0)
        r = torch.rand(b, 4, generator=host)
        kinds = [FILTERS[case["filter"]]] * b if case["filter"] in FILTERS else \
            [list(FILTERS.values())[i % 5] for i in range(b)]
        some_k, some_p, some_m = torch.tensor(kinds).t()
        temperature = 0.6 + 0.7 * r[:, 0]
        if case["filter"] == "mixed":
            temperature[2::6] = 0.0                          # greedy
        top_k = torch.where(some_k > 0, (5 * 100 ** r[:, 1]).long(), torch.zeros(b, dtype=torch.long))
        return {"logits": x.to(TORCH_DTYPE[case["dtype"]]), "u": torch.rand(b, generator=g, device=DEVICE),
                "temperature": temperature.to(DEVICE), "top_k": top_k.int().to(DEVICE),
                "top_p": torch.where(some_p > 0, torch.ones(b), 0.7 + 0.28 * r[:, 2]).to(DEVICE),
                "min_p": (some_m * (0.01 + 0.15 * r[:, 3])).to(DEVICE)}
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    seqs = shuffled(_sequences(case))
    need = [_pages_of(l, page) for _, l in seqs]
    first = _pages_of(case["prefix"], page)
    total = sum(need) + first + 7
    order = torch.randperm(total, generator=host).to(torch.int32)
    table, at = torch.zeros(len(seqs), max(need), dtype=torch.int32), first
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    start = [0]
    for n, _ in seqs:
        start.append(start[-1] + n)
    return {"q": normal(start[-1], hq, d, std=1.5), "k": normal(total, hkv, page, d), "v": normal(total, hkv, page, d),
            "prefix_pages": order[:first].to(DEVICE), "prefix_len": ints([case["prefix"]]), "pages": table.to(DEVICE),
            "start": ints(start), "len": ints([l for _, l in seqs]), "max_new": max(n for n, _ in seqs),
            "max_len": case["len_hi"], "max_prefix": case["prefix"]}


def prepare(case, seed):
    st = {"case": case, **_inputs(case, seed)}
    if own:
        st["call"] = _call(case, st)
    torch.cuda.synchronize()      # the library's stream is its own: the inputs are written
    return st


# ------------------------------------------------------------------- the library ---
def _call(case, t):
    """The operator's call with its arguments in hand: library headers over the program's
    tensors, its output buffers and parameters."""
    from onnx_translator_amd.nn import DTYPE_MAP, Ops
    from onnx_translator_amd.nn import Operators as operators
    lib = Ops._get_lib()
    name_of = {v: k for k, v in TORCH_DTYPE.items()}
    held = []

    def wrap(x):
        shape = tuple(x.shape)
        held.append(lib.tensor_wrap_device(ctypes.c_void_p(x.data_ptr()), (ctypes.c_int * len(shape))(*shape),
                                           len(shape), DTYPE_MAP[name_of[x.dtype]]))
        return held[-1]

    def empty(*shape, dtype=torch.int32):
        return torch.empty(*shape, dtype=dtype, device=DEVICE)

    if case["op"] == "plan":
        b, rows = case["b"], t["rows"]
        out = [empty(b + 1), empty(b), empty(rows), empty(rows), t["pages"], t["free"], torch.empty_like(t["state"])]
        start, length, positions, slots, pages, free, state = (wrap(x) for x in out)
        params = operators.CCachePlanParams(case["page"])
        args = [wrap(t["new"]), wrap(t["past"]), wrap(t["offset"]), wrap(t["state"]), pages, free, start, length,
                positions, slots, state, ctypes.byref(params)]
        fn, result = lib.cache_plan_forward, out
    elif case["op"] == "prefix":
        out = torch.empty_like(t["q"])
        params = operators.CPrefixAttentionParams(0.0, t["max_prefix"], t["max_len"])
        args = [wrap(t["q"]), wrap(t["k"]), wrap(t["v"]), wrap(t["prefix_pages"]), wrap(t["prefix_len"]),
                wrap(t["pages"]), wrap(t["start"]), wrap(t["len"]), wrap(out), ctypes.byref(params), None]
        fn, result = lib.prefix_cache_attention_forward, out
    else:
        out = [empty(case["b"]), empty(case["b"], dtype=torch.float32)]
        params = operators.CSampleParams(0)
        args = [wrap(t["logits"]), wrap(t["u"]), wrap(t["temperature"]), wrap(t["top_k"]), wrap(t["top_p"]),
                wrap(t["min_p"]), wrap(out[0]), wrap(out[1]), ctypes.byref(params), None]
        fn, result = lib.sample_forward, out
    return {"fn": fn, "args": args, "result": result, "error": lib.tensor_ops_hip_last_error, "held": (held, params)}


# ------------------------------------------------------------------------- call ---
def run(st):
    if own:
        call = st["call"]
        call["fn"](*call["args"])
        err = call["error"]()
        if err:
            raise RuntimeError(err.decode())
        return call["result"]
    return {"plan": _plan, "prefix": _prefix, "sample": _sample}[st["case"]["op"]](st)


def _plan(st):
    page, table, free, rows = st["case"]["page"], st["pages"], st["free"], st["rows"]
    new, past = st["new"].long(), st["past"].long()
    b, cols = table.shape
    size = free.numel()
    taken, returned = st["state"][0], st["state"][1]
    ended, n = new < 0, new.clamp(min=0)
    have = (past + page - 1) // page
    col = torch.arange(cols, device=DEVICE)
    # pages of ended requests go back to the ring
    back = torch.where(ended, have, torch.zeros_like(have))
    at = returned + (back.cumsum(0) - back)[:, None] + col
    at = torch.where(col < back[:, None], at % size, torch.full_like(at, size))
    free.copy_(torch.cat([free, free[:1]]).scatter_(0, at.reshape(-1), table.reshape(-1))[:size])
    returned = returned + back.sum()
    # the others take what their new tokens need, in order, as long as there are pages
    end = n.cumsum(0)
    fits = ~ended & (end <= rows) & ((past + n + page - 1) // page <= cols)
    need = torch.where(fits, (past + n + page - 1) // page - have, torch.zeros_like(have))
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= returned - taken))
    take = torch.where(served, need, torch.zeros_like(need))
    takes = (col >= have[:, None]) & (col < (have + take)[:, None])
    table.copy_(torch.where(takes, free[(taken + (upto - need - have)[:, None] + col) % size], table))
    start = torch.cat([torch.zeros_like(end[:1]), end]).clamp(max=rows)
    zero = torch.zeros_like(past)
    length = torch.where(ended, zero, torch.where(served, past + n, past))
    # positions and slots of the new tokens
    t = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(end, t, right=True)
    real = seq < b
    seq = seq.clamp(max=b - 1)
    real = real & served[seq]
    place = past[seq] + t - (end - n)[seq]
    none = torch.full_like(t, -1)
    positions = torch.where(real, place + st["offset"].long(), none)
    where = table[seq, torch.where(real, place // page, torch.zeros_like(t))].long()
    slots = torch.where(real, where * page + place % page, none)
    refused = (~ended & ~served).sum()
    state = torch.stack([taken + take.sum(), returned, refused])
    return [start.int(), length.int(), positions.int(), slots.int(), table, free, state]


def _gathered(cache, pages):
    """The pages of each sequence, one behind the other: [sequences, heads, keys, d] in float32."""
    b, most = pages.shape
    _, hkv, page, d = cache.shape
    return cache[pages.long()].permute(0, 2, 1, 3, 4).reshape(b, hkv, most * page, d).float()


def _prefix(st):
    case, q, start, lens = st["case"], st["q"], st["start"].long(), st["len"].long()
    tokens, hq, d = q.shape
    b, hkv, most = len(lens), case["hkv"], st["max_new"]
    group, shared = hq // hkv, case["prefix"]
    pk, pv = (_gathered(st[c], st["prefix_pages"][None])[0, :, :shared] for c in ("k", "v"))
    k, v = _gathered(st["k"], st["pages"]), _gathered(st["v"], st["pages"])
    scale = 1.0 / math.sqrt(d)
    # scores over the prefix: all tokens at once
    rows = q.float().reshape(tokens, hkv, group, d).permute(1, 0, 2, 3).reshape(hkv, tokens * group, d)
    s = torch.matmul(rows, pk.transpose(1, 2).contiguous()) * scale
    top = s.amax(-1, keepdim=True)
    # and over each sequence's own keys: its tokens padded to the longest chunk
    i = torch.arange(most, device=DEVICE)
    at = torch.clamp(start[:-1, None] + i, max=tokens - 1)
    own_rows = q.float()[at].reshape(b, most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, most * group, d)
    z = torch.matmul(own_rows, k.transpose(2, 3).contiguous()) * scale
    pos = (lens - (start[1:] - start[:-1]))[:, None] + i
    open_ = torch.arange(k.shape[2], device=DEVICE) <= pos[:, :, None]
    open_ = open_[:, None, :, None].expand(b, 1, most, group, -1).reshape(b, 1, most * group, -1)
    z = z.masked_fill(~open_, float("-inf"))
    # both to the order of the tokens, joined by their largest scores
    t = torch.arange(tokens, device=DEVICE)
    seq = torch.searchsorted(start[1:].contiguous(), t, right=True)
    place = t - start[seq]

    def of_tokens(x):
        x = x.reshape(b, hkv, most, group, -1)[seq, :, place]
        return x.permute(1, 0, 2, 3).reshape(hkv, tokens * group, -1)

    own_top = z.amax(-1, keepdim=True)
    m = torch.maximum(top, of_tokens(own_top))
    padded = torch.zeros(b, most, hkv, group, 1, device=DEVICE)
    padded[seq, place] = m.reshape(hkv, tokens, group, 1).permute(1, 0, 2, 3)
    p = torch.exp(s - m)
    w = torch.exp(z - padded.permute(0, 2, 1, 3, 4).reshape(b, hkv, most * group, 1))
    total = p.sum(-1, keepdim=True) + of_tokens(w.sum(-1, keepdim=True))
    o = (torch.matmul(p, pv) + of_tokens(torch.matmul(w, v))) / total
    return o.reshape(hkv, tokens, group, d).permute(1, 0, 2, 3).reshape(tokens, hq, d).to(q.dtype)


def _sample(st):
    x = st["logits"].double()
    b, v = x.shape
    t, p, low = (st[c].double()[:, None] for c in ("temperature", "top_p", "min_p"))
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = t <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    rank = torch.arange(v, device=DEVICE)
    k = st["top_k"].long()[:, None]
    k = torch.where(k > 0, k, torch.full_like(k, v))
    k = torch.where(greedy, torch.ones_like(k), k)
    w = torch.where(rank < k, w, torch.zeros_like(w))
    upto = w.cumsum(1)
    kept = ((upto - w < p * upto[:, -1:]) | (p >= 1) | (rank == 0)) & (w >= low) & (rank < k)
    w = torch.where(kept, w, torch.zeros_like(w))
    # drawn in the order of the tokens
    w = torch.zeros_like(w).scatter_(1, order, w)
    upto = w.cumsum(1)
    total = upto[:, -1:]
    token = (upto <= st["u"].double()[:, None] * total).sum(1, keepdim=True)
    last = (torch.arange(v, device=DEVICE) * (w > 0)).amax(1, keepdim=True)
    token = torch.minimum(token, last)
    chance = torch.log(w.gather(1, token) / total)
    return [token[:, 0].int(), chance[:, 0].float()]


# ---------------------------------------------------------------------- 64 bits ---
def _exact_plan(case, t):
    new, past, table, free, state = (t[c].cpu().numpy().astype(np.int64) for c in ("new", "past", "pages", "free", "state"))
    page, rows, size, offset = case["page"], t["rows"], len(free), int(t["offset"][0])
    taken, returned = int(state[0]), int(state[1])
    for i in np.flatnonzero(new < 0):
        n = _pages_of(int(past[i]), page)
        free[(returned + np.arange(n)) % size] = table[i, :n]
        returned += n
    start, length = [0], []
    positions, slots = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    asked = refused = 0
    spare = returned - taken
    for i in range(len(new)):
        n, l = max(int(new[i]), 0), int(past[i])
        begin = start[-1]
        start.append(min(begin + n, rows))
        if new[i] < 0:
            length.append(0)
            continue
        have, most = _pages_of(l, page), _pages_of(l + n, page)
        fits = begin + n <= rows and most <= table.shape[1]
        if fits:
            asked += most - have
        if not fits or (most > have and asked > spare):
            refused += 1
            length.append(l)
            continue
        table[i, have:most] = free[(taken + np.arange(most - have)) % size]
        taken += most - have
        at = l + np.arange(n)
        positions[begin:begin + n] = at + offset
        slots[begin:begin + n] = table[i, at // page] * page + at % page
        length.append(l + n)
    return [np.array(x, np.int64) for x in (start, length, positions, slots, table, free, [taken, returned, refused])]


def _exact_prefix(case, t):
    q, page, group, d = t["q"], case["page"], case["hq"] // case["hkv"], case["d"]
    out = torch.empty(q.shape, dtype=torch.float64, device=DEVICE)
    start, lens = t["start"].tolist(), t["len"].tolist()
    for h in range(case["hkv"]):
        pk, pv = (t[c][t["prefix_pages"].long(), h].reshape(-1, d)[:case["prefix"]].double() for c in ("k", "v"))
        for i, m in enumerate(lens):
            which = t["pages"][i, :_pages_of(m, page)].long()
            k, v = (torch.cat([c, t[n][which, h].reshape(-1, d)[:m].double()]) for n, c in (("k", pk), ("v", pv)))
            n = start[i + 1] - start[i]
            pos = case["prefix"] + torch.arange(m - n, m, device=DEVICE)[:, None]
            unseen = torch.arange(len(k), device=DEVICE)[None] > pos
            kt = k.t().contiguous() / math.sqrt(d)
            for j in range(h * group, (h + 1) * group):
                s = q[start[i]:start[i + 1], j].double() @ kt
                out[start[i]:start[i + 1], j] = torch.softmax(s.masked_fill(unseen, -math.inf), 1) @ v
    return out


def _exact_sample(case, t):
    tokens, chances = [], []
    settings = [t[c].double().tolist() for c in ("temperature", "top_p", "min_p", "top_k", "u")]
    for row, temp, p, low, k, u in zip(t["logits"], *settings):
        x = row.double()
        if temp <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            chances.append(0.0)
            continue
        x = (x - x.max()) / temp
        # rank by value, equal ones by place
        ranked = torch.argsort(-x, stable=True)
        ranked = ranked[:int(k)] if k > 0 else ranked
        w = x[ranked].exp()
        if p < 1:
            mass = w.cumsum(0)
            ranked = ranked[:max(1, int((torch.cat([mass.new_zeros(1), mass[:-1]]) < p * mass[-1]).sum()))]
        ranked = ranked[x[ranked].exp() >= low]
        places = ranked.sort()[0]
        mass = x[places].exp().cumsum(0)
        at = min(int(torch.searchsorted(mass, u * mass[-1], right=True)), len(places) - 1)
        tokens.append(int(places[at]))
        chances.append(float(x[places[at]] - mass[-1].log()))
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(chances, dtype=torch.float64)]


def exact(case, seed):
    t = _inputs(case, seed)
    return {"plan": _exact_plan, "prefix": _exact_prefix, "sample": _exact_sample}[case["op"]](case, t)
