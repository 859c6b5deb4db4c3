"""The attention path of a decoder layer, as cases that can be timed and compared.

Three operators, between the projection Gemms of a layer:

* ``rotary``: per-head RMS norm of queries and keys, rotation by position, keys and values
  into the pages of a cache or into dense tensors (``qk_norm_rotary_forward``);
* ``cache``: a chunk of new tokens of each sequence over its paged cache
  (``cache_attention_forward``), single tokens and prompts alike;
* ``attn``: attention to keys and values of another length, with masks and lengths
  (``attention_forward``).

A case is a dict of plain values.  ``listed()`` names twelve, ``draw(rng)`` gives more of the
same ranges.  ``prepare`` makes what a program holds before the call, ``run`` makes the call:
elementary torch operations in float32 where ``own`` is false, the library's operators where it
is true.  ``exact`` restates the operator in 64 bits.
"""
import ctypes
import math

import torch

own = False

DEVICE = "cuda"
TORCH_DTYPE = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
               "int32": torch.int32, "uint8": torch.uint8}
ELEM_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
EPSILON = 1e-6


def listed():
    return [
        # One token of one request over an encoder's states: the smallest attention a decoder
        # asks for, where the launch counts as much as the 6 MB.
        {"name": "attn_one_token", "op": "attn", "b": 1, "sq": 1, "skv": 1500, "hq": 16, "hkv": 16, "d": 64,
         "dtype": "float16", "mask": "none", "causal": False},
        # The same step for a batch of requests whose encoder inputs have different lengths.
        {"name": "attn_tokens_lengths", "op": "attn", "b": 32, "sq": 1, "skv": 1500, "hq": 16, "hkv": 16, "d": 64,
         "dtype": "float16", "mask": "lengths", "causal": False},
        # A decoder's whole prompt over padded encoder states: neither length fills its tiles.
        {"name": "attn_cross_lengths", "op": "attn", "b": 8, "sq": 448, "skv": 1500, "hq": 16, "hkv": 16, "d": 64,
         "dtype": "float16", "mask": "lengths", "causal": False},
        # An exported float32 graph: odd lengths, an additive mask per batch.
        {"name": "attn_mask_f32", "op": "attn", "b": 4, "sq": 197, "skv": 577, "hq": 12, "hkv": 12, "d": 64,
         "dtype": "float32", "mask": "additive", "causal": False},
        # Long states, shared key heads: bound by the matrix cores.
        {"name": "attn_long", "op": "attn", "b": 1, "sq": 4096, "skv": 8192, "hq": 32, "hkv": 8, "d": 128,
         "dtype": "bfloat16", "mask": "none", "causal": False},
        # One token of one conversation: latency.
        {"name": "cache_one_token", "op": "cache", "b": 1, "n_lo": 1, "n_hi": 1, "len_lo": 1025, "len_hi": 1025,
         "hq": 32, "hkv": 8, "d": 128, "page": 16, "window": 0, "dtype": "bfloat16"},
        # A decoding batch at all ages up to 8192 tokens: what serving spends its time on.
        {"name": "cache_tokens", "op": "cache", "b": 64, "n_lo": 1, "n_hi": 1, "len_lo": 130, "len_hi": 8192,
         "hq": 32, "hkv": 8, "d": 128, "page": 16, "window": 0, "dtype": "bfloat16"},
        # Decoding requests and prompt chunks in one batch, groups of three heads, pages of 32.
        {"name": "cache_mixed", "op": "cache", "b": 12, "n_lo": 1, "n_hi": 512, "len_lo": 513, "len_hi": 4000,
         "hq": 24, "hkv": 8, "d": 64, "page": 32, "window": 0, "dtype": "float16"},
        # A chunk of a long prompt behind what is cached of it.
        {"name": "cache_prompt_chunk", "op": "cache", "b": 1, "n_lo": 4096, "n_hi": 4096, "len_lo": 16384,
         "len_hi": 16384, "hq": 32, "hkv": 8, "d": 128, "page": 16, "window": 0, "dtype": "bfloat16"},
        # The tokens of a small decoding batch on their way into the cache: latency.
        {"name": "rotary_tokens", "op": "rotary", "t": 8, "hq": 32, "hkv": 8, "d": 128, "r": 128,
         "interleaved": False, "norm": True, "page": 16, "dtype": "bfloat16"},
        # A prompt's projections into the cache: bound by memory.
        {"name": "rotary_prompt", "op": "rotary", "t": 8192, "hq": 32, "hkv": 8, "d": 128, "r": 128,
         "interleaved": False, "norm": True, "page": 16, "dtype": "bfloat16"},
        # Part of each head rotated, pairs interleaved, dense outputs, an odd number of tokens.
        {"name": "rotary_partial_f32", "op": "rotary", "t": 1023, "hq": 12, "hkv": 4, "d": 80, "r": 40,
         "interleaved": True, "norm": True, "page": 0, "dtype": "float32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "cache", "cache", "rotary"])
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    hkv = rng.choice([1, 2, 4, 5, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8]) if hkv <= 8 else 1
    d = rng.choice([64, 64, 128, 128, 128, 32, 40, 80, 96, 192, 256])
    case = {"op": op, "hq": hkv * group, "hkv": hkv, "d": d, "dtype": dtype}
    most = 4e11 if dtype != "float32" else 4e10             # operations of a pass
    if op == "attn":
        case.update(b=_log(rng, 1, 48), sq=1 if rng.random() < 0.3 else _log(rng, 2, 4096), skv=_log(rng, 1, 8192),
                    mask=rng.choice(["none", "lengths", "additive", "bool"]), causal=rng.random() < 0.2)
        while case["b"] > 1 and work(case)["flops"] > most:
            case["b"] = (case["b"] + 1) // 2
        while work(case)["flops"] > most:
            case["sq"] = (case["sq"] + 1) // 2
    elif op == "cache":
        hi = _log(rng, 1, 16384)
        n_hi = 1 if rng.random() < 0.4 else _log(rng, 1, min(hi, 4096))
        case.update(b=_log(rng, 1, 64), n_lo=1 if rng.random() < 0.6 else n_hi, n_hi=n_hi,
                    len_lo=rng.randint(max(1, n_hi), hi), len_hi=hi, page=rng.choice([16, 16, 32, 64, 128, 24]),
                    window=rng.choice([0, 0, 0, 128, 1000]))
        while case["b"] > 1 and (work(case)["flops"] > most or
                                 case["b"] * case["hq"] * case["n_hi"] * case["len_hi"] > 1 << 31 or
                                 case["b"] * case["hkv"] * case["len_hi"] * d > 1 << 30):
            case["b"] = (case["b"] + 1) // 2
        while work(case)["flops"] > most:
            case["n_hi"] = (case["n_hi"] + 1) // 2
            case["n_lo"] = min(case["n_lo"], case["n_hi"])
    else:
        case.update(t=_log(rng, 1, 8192), r=rng.choice([d, d, d // 2, 16]), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.8, page=rng.choice([16, 64, 0]))
        while case["t"] > 1 and case["t"] * (case["hq"] + 2 * hkv) * d > 1 << 26:
            case["t"] //= 2
    return case


# ------------------------------------------------------------------------ sizes ---
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _sequences(case):
    """(new tokens, length) of each sequence: the longest chunk in the middle of the lengths,
    single tokens around it."""
    b = case["b"]
    lens = _spread(case["len_lo"], case["len_hi"], b)
    lo, hi = case["n_lo"], case["n_hi"]
    news = [max(lo, int(round(hi ** (1 - abs(2 * i - b + 1) / max(b, 2))))) if hi > lo else hi for i in range(b)]
    return [(min(n, l), l) for n, l in zip(news, lens)]


def _seen(first, n, window):
    """Keys seen by n tokens from position `first` on, together."""
    if not window or first + n <= window:
        return n * first + n * (n + 1) // 2
    return sum(min(first + i + 1, window) for i in range(n))


def work(case):
    e, hq, hkv, d = ELEM_BYTES[case["dtype"]], case["hq"], case["hkv"], case["d"]
    if case["op"] == "rotary":
        values = case["t"] * (hq + 2 * hkv) * d
        return {"bytes": 2 * values * e + 4 * case["t"] * (case["r"] + 2), "flops": 8 * values}
    if case["op"] == "attn":
        b, sq, skv = case["b"], case["sq"], case["skv"]
        lens = _lengths(case)
        pairs = sum(sum(min(i + 1, l) for i in range(sq)) if case["causal"] else sq * l for l in lens)
        mask = {"additive": e * b * sq * skv, "bool": b * sq * skv}.get(case["mask"], 0)
        return {"bytes": e * d * (2 * b * sq * hq + 2 * sum(lens) * hkv) + mask, "flops": 4 * d * hq * pairs}
    seqs = _sequences(case)
    pairs = sum(_seen(l - n, n, case["window"]) for n, l in seqs)
    read = sum(min(l, n + case["window"]) if case["window"] else l for n, l in seqs)
    return {"bytes": e * d * (2 * sum(n for n, _ in seqs) * hq + 2 * read * hkv), "flops": 4 * d * hq * pairs}


def _lengths(case):
    """Keys in use per batch."""
    if case["mask"] != "lengths":
        return [case["skv"]] * case["b"]
    return _spread(max(1, case["skv"] // 5), case["skv"], case["b"])


# ----------------------------------------------------------------------- inputs ---
def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    host = torch.Generator()
    host.manual_seed(int(seed))
    dt, hq, hkv, d = TORCH_DTYPE[case["dtype"]], case["hq"], case["hkv"], case["d"]

    def normal(*shape, std=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dtype or dt)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEVICE)

    if case["op"] == "attn":
        b, sq, skv = case["b"], case["sq"], case["skv"]
        t = {"q": normal(b, hq, sq, d, std=1.5), "k": normal(b, hkv, skv, d), "v": normal(b, hkv, skv, d)}
        if case["mask"] == "lengths":
            lens = _lengths(case)
            t["len"] = ints([lens[i] for i in torch.randperm(b, generator=host).tolist()])
        elif case["mask"] == "additive":
            # a bias by distance, and one key in eight closed to a query
            t["mask"] = normal(b, 1, sq, skv, std=0.5)
            t["mask"][torch.rand(b, 1, sq, skv, generator=g, device=DEVICE) < 0.125] = float("-inf")
        elif case["mask"] == "bool":
            t["mask"] = (torch.rand(b, 1, sq, skv, generator=g, device=DEVICE) < 0.875).to(torch.uint8)
        return t
    if case["op"] == "cache":
        seqs = _sequences(case)
        seqs = [seqs[i] for i in torch.randperm(len(seqs), generator=host).tolist()]
        page = case["page"]
        need = [-(-l // page) for _, l in seqs]
        most = max(need)
        total = sum(need) + 7
        order = torch.randperm(total, generator=host)
        table, at = torch.zeros(len(seqs), most, dtype=torch.int32), 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n].to(torch.int32)
            at += n
        start = [0]
        for n, _ in seqs:
            start.append(start[-1] + n)
        return {"q": normal(start[-1], hq, d, std=1.5), "k": normal(total, hkv, page, d),
                "v": normal(total, hkv, page, d), "pages": table.to(DEVICE), "start": ints(start),
                "len": ints([l for _, l in seqs]), "max_new": max(n for n, _ in seqs), "max_len": case["len_hi"]}
    tokens, r, page = case["t"], case["r"], case["page"]
    t = {"qkv": normal(tokens, (hq + 2 * hkv) * d, std=2.0)}
    if case["norm"]:
        t["wq"], t["wk"] = normal(d, std=0.1) + 1, normal(d, std=0.1) + 1
    rows = 4 * tokens + 4096
    angle = (torch.arange(rows, dtype=torch.float64, device=DEVICE)[:, None] *
             10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEVICE) / r))
    t["cos"], t["sin"] = angle.cos().float(), angle.sin().float()
    t["pos"] = (torch.arange(tokens, device=DEVICE) + torch.randint(0, rows - tokens, (1,), generator=host).item()).int()
    if page:
        pages = -(-tokens // page) + 5
        t["k"], t["v"] = normal(pages, hkv, page, d), normal(pages, hkv, page, d)
        order = torch.randperm(pages, generator=host).to(DEVICE)
        at = torch.arange(tokens, device=DEVICE)
        t["slots"] = (order[at // page] * page + at % page).int()
    return t


def prepare(case, seed):
    st = {"case": case, **_inputs(case, seed)}
    if own:
        st["call"] = _call(case, st)
    torch.cuda.synchronize()      # the library's stream is its own: the inputs are written
    return st


# ------------------------------------------------------------------- the library ---
def _call(case, t):
    """The operator's call with its arguments in hand: library headers over the program's
    tensors, its output buffers and a workspace."""
    from onnx_translator_amd.nn import DTYPE_MAP, Ops
    from onnx_translator_amd.nn import Operators as operators
    lib = Ops._get_lib()
    name_of = {v: k for k, v in TORCH_DTYPE.items()}
    held = []

    def wrap(x):
        if x is None:
            return None
        shape = tuple(x.shape)
        held.append(lib.tensor_wrap_device(ctypes.c_void_p(x.data_ptr()), (ctypes.c_int * len(shape))(*shape),
                                           len(shape), DTYPE_MAP[name_of[x.dtype]]))
        return held[-1]

    dt = TORCH_DTYPE[case["dtype"]]
    if case["op"] == "attn":
        out = torch.empty(case["b"], case["hq"], case["sq"], case["d"], dtype=dt, device=DEVICE)
        params = operators.CAttentionParams(0, 0, 0.0, int(case["causal"]))
        args = [wrap(t["q"]), wrap(t["k"]), wrap(t["v"]), wrap(t.get("mask")), wrap(t.get("len")), wrap(out),
                ctypes.byref(params), None]
        fn, result = lib.attention_forward, out
    elif case["op"] == "cache":
        out = torch.empty_like(t["q"])
        params = operators.CCacheAttentionParams(0.0, case["window"], t["max_len"])
        args = [wrap(t["q"]), wrap(t["k"]), wrap(t["v"]), wrap(t["pages"]), wrap(t["start"]), wrap(t["len"]),
                wrap(out), ctypes.byref(params), None]
        fn, result = lib.cache_attention_forward, out
    else:
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        q = torch.empty(case["t"], hq, d, dtype=dt, device=DEVICE)
        if case["page"]:
            k, v = t["k"], t["v"]
        else:
            k, v = (torch.empty(case["t"], hkv, d, dtype=dt, device=DEVICE) for _ in range(2))
        params = operators.CQKNormRotaryParams(hq, hkv, EPSILON, int(case["interleaved"]))
        args = [wrap(t["qkv"]), wrap(t.get("wq")), wrap(t.get("wk")), wrap(t["cos"]), wrap(t["sin"]), wrap(t["pos"]),
                wrap(t.get("slots")), wrap(q), wrap(k), wrap(v), ctypes.byref(params)]
        fn, result = lib.qk_norm_rotary_forward, [q, k, v]
    return {"fn": fn, "args": args, "result": result, "error": lib.tensor_ops_hip_last_error,
            "held": (held, params)}


# ------------------------------------------------------------------------- call ---
def run(st):
    if own:
        call = st["call"]
        call["fn"](*call["args"])
        err = call["error"]()
        if err:
            raise RuntimeError(err.decode())
        return call["result"]
    return {"attn": _attn, "cache": _cache, "rotary": _rotary}[st["case"]["op"]](st)


def _weights(s, open_):
    """Softmax of the scores over the open keys; a row without any gives zeros."""
    if open_ is not None:
        s = s.masked_fill(~open_, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _attn(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    b, hq, sq, d = q.shape
    hkv, skv = k.shape[1:3]
    group = hq // hkv
    s = torch.matmul(q.float().reshape(b, hkv, group * sq, d), k.float().transpose(2, 3).contiguous())
    s = (s / math.sqrt(d)).reshape(b, hq, sq, skv)
    open_ = None
    key = torch.arange(skv, device=DEVICE)
    if case["mask"] == "lengths":
        open_ = (key < st["len"][:, None])[:, None, None]
    elif case["mask"] == "additive":
        s = s + st["mask"].float()
    elif case["mask"] == "bool":
        open_ = st["mask"] != 0
    if case["causal"]:
        below = key <= torch.arange(sq, device=DEVICE)[:, None]
        open_ = below if open_ is None else open_ & below
    p = _weights(s, open_).reshape(b, hkv, group * sq, skv)
    return torch.matmul(p, v.float()).reshape(b, hq, sq, d).to(q.dtype)


def _gathered(cache, pages):
    """The pages of each sequence, one behind the other: [sequences, heads, keys, d] in float32."""
    b, most = pages.shape
    _, hkv, page, d = cache.shape
    return cache[pages.long()].permute(0, 2, 1, 3, 4).reshape(b, hkv, most * page, d).float()


def _cache(st):
    case, q, start, lens = st["case"], st["q"], st["start"].long(), st["len"].long()
    tokens, hq, d = q.shape
    b, hkv, most = len(lens), case["hkv"], st["max_new"]
    group = hq // hkv
    k, v = _gathered(st["k"], st["pages"]), _gathered(st["v"], st["pages"])
    # the new tokens of each sequence, padded to the longest chunk
    i = torch.arange(most, device=DEVICE)
    at = torch.clamp(start[:-1, None] + i, max=tokens - 1)
    rows = q.float()[at].reshape(b, most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, most * group, d)
    s = torch.matmul(rows, k.transpose(2, 3).contiguous()) / math.sqrt(d)
    pos = (lens - (start[1:] - start[:-1]))[:, None] + i
    key = torch.arange(k.shape[2], device=DEVICE)
    open_ = key <= pos[:, :, None]
    if case["window"]:
        open_ = open_ & (key > pos[:, :, None] - case["window"])
    open_ = open_[:, None, :, None].expand(b, 1, most, group, -1).reshape(b, 1, most * group, -1)
    o = torch.matmul(_weights(s, open_), v).reshape(b, hkv, most, group, d)
    # back to the order of the tokens
    t = torch.arange(tokens, device=DEVICE)
    seq = torch.searchsorted(start[1:].contiguous(), t, right=True)
    return o[seq, :, t - start[seq]].reshape(tokens, hq, d).to(q.dtype)


def _rotary(st):
    case, qkv = st["case"], st["qkv"]
    tokens, hq, hkv, d, r = qkv.shape[0], case["hq"], case["hkv"], case["d"], case["r"]
    x = qkv.reshape(tokens, hq + 2 * hkv, d)
    h = x[:, :hq + hkv].float()
    if case["norm"]:
        w = torch.cat([st["wq"].float().expand(hq, d), st["wk"].float().expand(hkv, d)])
        h = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPSILON) * w
    c, s = st["cos"][st["pos"].long()][:, None], st["sin"][st["pos"].long()][:, None]
    if case["interleaved"]:
        a, b = h[..., 0:r:2], h[..., 1:r:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).reshape(tokens, hq + hkv, r)
    else:
        a, b = h[..., :r // 2], h[..., r // 2:r]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    h = torch.cat([turned, h[..., r:]], -1).to(qkv.dtype)
    q, k, v = h[:, :hq].contiguous(), h[:, hq:], x[:, hq + hkv:]
    if not case["page"]:
        return [q, k.contiguous(), v.contiguous()]
    page = case["page"]
    slot = st["slots"].long()
    st["k"][slot // page, :, slot % page] = k
    st["v"][slot // page, :, slot % page] = v
    return [q, st["k"], st["v"]]


# ---------------------------------------------------------------------- 64 bits ---
def _rows64(q, k, v, seen, bias=None):
    """Attention of the rows q [n, d] over k, v [m, d]: seen (truth values [n, m]) and bias."""
    s = q.double() @ k.double().t().contiguous() * (1.0 / math.sqrt(q.shape[1]))
    if bias is not None:
        s = s + bias.double()
    if seen is not None:
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
    none = ~torch.isfinite(s).any(1, keepdim=True)
    p = torch.softmax(torch.where(none, torch.zeros_like(s), s), 1)
    return torch.where(none, torch.zeros_like(p), p) @ v.double()


def _exact_attn(case, t):
    q, k, v = t["q"], t["k"], t["v"]
    b, hq, sq, d = q.shape
    skv, group = case["skv"], hq // case["hkv"]
    out = torch.empty(b, hq, sq, d, dtype=torch.float64, device=DEVICE)
    lens = t["len"].tolist() if "len" in t else [skv] * b
    below = torch.ones(sq, skv, dtype=torch.bool, device=DEVICE).tril() if case["causal"] else None
    for i in range(b):
        m = lens[i]
        seen, bias = (below[:, :m] if below is not None else None), None
        if case["mask"] == "additive":
            bias = t["mask"][i, 0]
        elif case["mask"] == "bool":
            seen = t["mask"][i, 0] != 0 if seen is None else seen & (t["mask"][i, 0] != 0)
        for h in range(hq):
            out[i, h] = _rows64(q[i, h], k[i, h // group, :m], v[i, h // group, :m], seen, bias)
    return out


def _exact_cache(case, t):
    q, page, group = t["q"], case["page"], case["hq"] // case["hkv"]
    out = torch.empty(q.shape, dtype=torch.float64, device=DEVICE)
    start, lens = t["start"].tolist(), t["len"].tolist()
    for i, m in enumerate(lens):
        n = start[i + 1] - start[i]
        which = t["pages"][i, :-(-m // page)].long()
        pos = torch.arange(m - n, m, device=DEVICE)[:, None]
        key = torch.arange(m, device=DEVICE)[None]
        seen = key <= pos
        if case["window"]:
            seen &= key > pos - case["window"]
        for h in range(case["hkv"]):
            k, v = (t[c][which, h].reshape(-1, case["d"])[:m] for c in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                out[start[i]:start[i + 1], j] = _rows64(q[start[i]:start[i + 1], j], k, v, seen)
    return out


def _exact_rotary(case, t):
    tokens, hq, hkv, d, r = case["t"], case["hq"], case["hkv"], case["d"], case["r"]
    q, k, v = t["qkv"].reshape(tokens, -1, d).split([hq, hkv, hkv], 1)
    pos = t["pos"].long()
    # a pair is a complex number, its rotation a product
    turn = torch.complex(t["cos"][pos].double(), t["sin"][pos].double())[:, None]

    def head(x, w):
        x = x.double()
        if case["norm"]:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPSILON) * t[w].double()
        x = x.clone()
        pair = (x[..., :r].unflatten(-1, (r // 2, 2)) if case["interleaved"] else
                x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2))
        z = torch.view_as_real(torch.complex(pair[..., 0].contiguous(), pair[..., 1].contiguous()) * turn)
        x[..., :r] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return x

    new = [head(q, "wq"), head(k, "wk"), v.double()]
    if not case["page"]:
        return new
    flat = t["slots"].long()
    for i, name in ((1, "k"), (2, "v")):
        cache = t[name].double()
        cache[flat // case["page"], :, flat % case["page"]] = new[i]
        new[i] = cache
    return new


def exact(case, seed):
    t = _inputs(case, seed)
    return {"attn": _exact_attn, "cache": _exact_cache, "rotary": _exact_rotary}[case["op"]](case, t)
