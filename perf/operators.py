"""The 8-bit key / value cache of ragged-batch serving and what reads it, as cases that can be timed and checked.

  write   a step's keys and values are quantised into their pages, a scale per token and head
  read    rows of one sequence come back as bfloat16 or float32
  attn    attention over the cache under a sliding window with a few first tokens that stay visible: single tokens, portions, both in one step
  tree    attention of drafted tokens over the cache and their own ancestors
  keep    the rows of an accepted path move to the front of the drafted ones, in all layers

  own (set by whoever imports this)   False: elementary torch operations; True: the calls that a program makes of krasis_b200
  listed() / draw(rng)                the cases; prepare(case, seed) / run(state) one pass; work(case) what it cannot do without;
  exact(case, seed)                   the same from the definition in 64 bits

Formats, per row (one token, one head) with largest magnitude a:
  e4m3   scale 2^k, the least with a <= 448 2^k;      int8   scale a / 127 in fp32;      codes are the nearest ones to number / scale, ties to even
"""
import math

import torch

own = False

DEV = "cuda:0"
BF = torch.bfloat16
PAGE = 64                                    # tokens a page, as the serving models have it
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _attn(name, seqs, lo, hi, n_lo, n_hi, heads, dims, fmt, window, first, q, out):
    """seqs sequences with lo .. hi rows cached before the step (spread evenly over the logarithm) that bring n_lo .. n_hi tokens each."""
    c = {"op": "attn", "seqs": seqs, "lo": lo, "hi": hi, "n_lo": n_lo, "n_hi": n_hi, "H": heads[0], "G": heads[1], "d": dims[0], "dv": dims[1], "fmt": fmt,
         "window": window, "first": first, "q": q, "out": out}
    return {"name": name, **c} if name else c


def listed():
    return [
        # four requests decode: one token each in one layer of the serving benchmark's geometry
        {"name": "write_decode", "op": "write", "seqs": 4, "lo": 100, "hi": 2048, "n_lo": 1, "n_hi": 1, "H": 16, "G": 2, "d": 128, "dv": 128, "fmt": "e4m3",
         "x": "float32"},
        # a long prompt's keys and values in one step, heads of the largest preset
        {"name": "write_prompt", "op": "write", "seqs": 1, "lo": 0, "hi": 0, "n_lo": 8192, "n_hi": 8192, "H": 64, "G": 4, "d": 128, "dv": 128, "fmt": "int8",
         "x": "bfloat16"},
        # the window of a short sequence comes back for a kernel that takes plain rows
        {"name": "read_window", "op": "read", "rows": 1027, "first": 301, "G": 2, "d": 128, "dv": 128, "fmt": "int8", "out": "bfloat16"},
        # a long sequence is read back whole (handed to another process, or checked)
        {"name": "read_context", "op": "read", "rows": 40001, "first": 0, "G": 4, "d": 128, "dv": 128, "fmt": "e4m3", "out": "bfloat16"},
        # four requests decode under a window of 1024 with four first tokens: latency
        _attn("attn_decode_few", 4, 700, 2048, 1, 1, (16, 2), (128, 128), "e4m3", 1024, 4, "float32", "bfloat16"),
        # a full batch of requests of very different lengths decodes without a window: memory
        _attn("attn_decode_many", 64, 500, 60000, 1, 1, (64, 4), (128, 128), "int8", 0, 0, "bfloat16", "bfloat16"),
        # a portion of a long prompt behind what is cached, under a window of 4096 with sixteen first tokens: tensor cores
        _attn("attn_portion", 1, 5001, 5001, 4096, 4096, (64, 4), (128, 128), "e4m3", 4096, 16, "float32", "bfloat16"),
        # a mixed step of the fp32 mode on heads of 256: portions of ragged length and single tokens
        _attn("attn_mixed_fp32", 6, 90, 3000, 1, 150, (16, 2), (256, 256), "int8", 0, 0, "float32", "float32"),
        # sixteen drafted tokens of one request are verified
        {"name": "tree_few", "op": "tree", "seqs": 1, "lo": 2001, "hi": 2001, "n_lo": 16, "n_hi": 16, "H": 16, "G": 2, "d": 128, "dv": 128, "fmt": "e4m3",
         "window": 0, "first": 0, "q": "float32", "out": "bfloat16", "span": 4},
        # sixteen requests with sixty-odd drafted tokens each behind long contexts
        {"name": "tree_many", "op": "tree", "seqs": 16, "lo": 2000, "hi": 30000, "n_lo": 57, "n_hi": 64, "H": 64, "G": 4, "d": 128, "dv": 128, "fmt": "int8",
         "window": 0, "first": 0, "q": "bfloat16", "out": "bfloat16", "span": 6},
        # the accepted path of one request in the six layer runs of the serving benchmark
        {"name": "keep_few", "op": "keep", "seqs": 1, "lo": 2001, "hi": 2001, "n_lo": 16, "n_hi": 16, "path": 4, "layers": 6, "H": 16, "G": 2, "d": 128, "dv": 128,
         "fmt": "e4m3"},
        # a full batch's paths in the layers of a large model
        {"name": "keep_many", "op": "keep", "seqs": 64, "lo": 100, "hi": 1500, "n_lo": 20, "n_hi": 64, "path": 8, "layers": 48, "H": 64, "G": 4, "d": 128, "dv": 128,
         "fmt": "int8"},
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attn", "attn", "attn", "attn", "tree", "tree", "tree", "keep"])
    H, G = rng.choice([(16, 2), (64, 4), (8, 8), (24, 8), (14, 2), (32, 1), (32, 4)])
    d, dv = rng.choice([(128, 128), (128, 128), (64, 64), (256, 256), (96, 96), (192, 128), (128, 256)])
    fmt = rng.choice(["e4m3", "int8"])
    q, out = rng.choice([("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("bfloat16", "bfloat16"), ("float32", "float32")])
    shape = {"H": H, "G": G, "d": d, "dv": dv, "fmt": fmt}
    window, first = rng.choice([(0, 0), (_logint(rng, 16, 6000), rng.choice([0, 1, 4, 37, 128]))])
    if op == "write":
        seqs = _logint(rng, 1, 16)
        n = _logint(rng, 1, 8192 // seqs)
        return {"op": op, "seqs": seqs, "lo": 0, "hi": _logint(rng, 1, 3000), "n_lo": 1 + n // 3, "n_hi": n, **shape, "x": q}
    if op == "read":
        return {"op": op, "rows": _logint(rng, 1, 40000), "first": rng.choice([0, _logint(rng, 1, 2000)]), **{k: shape[k] for k in ("G", "d", "dv", "fmt")}, "out": out}
    if op == "keep":
        n = _logint(rng, 2, 64)
        return {"op": op, "seqs": _logint(rng, 1, 64), "lo": 10, "hi": _logint(rng, 11, 1500), "n_lo": 1 + n // 2, "n_hi": n, "path": rng.randint(1, 1 + n // 2),
                "layers": rng.randint(1, 16), **shape}
    if op == "tree":
        seqs = _logint(rng, 1, 12)
        n = _logint(rng, 1, 64)
        lo = _logint(rng, 1, 4000)
        return {"op": op, "seqs": seqs, "lo": lo, "hi": max(lo, _logint(rng, 1, 16000)), "n_lo": 1 + n // 2, "n_hi": n, **shape, "window": window, "first": first, "q": q,
                "out": out, "span": rng.randint(1, 8)}
    if rng.random() < 0.6:                   # a step of decoded tokens
        seqs, lo = _logint(rng, 1, 64), _logint(rng, 1, 4000)
        return _attn(None, seqs, lo, max(lo, _logint(rng, 1, 30000)), 1, 1, (H, G), (d, dv), fmt, window, first, q, out)
    n = _logint(rng, 2, 1500)
    lo = rng.choice([0, _logint(rng, 1, 2000)])
    return _attn(None, rng.randint(1, 4), lo, lo + rng.choice([0, _logint(rng, 1, 3000)]), rng.choice([1, n]), n, (H, G), (d, dv), fmt, window, first, q, out)


# ------------------------------------------------------------------------------------------------ sizes that follow from a case

def _spread(lo, hi, count):
    """`count` numbers from lo to hi, evenly over the logarithm; one alone is hi."""
    if count == 1 or lo == hi:
        return [hi] * count
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * i / (count - 1)))) - 1 for i in range(count)]


def _lengths(case):
    """(rows cached before, tokens of the step) of every sequence: the longest contexts bring the fewest tokens."""
    return list(zip(_spread(case["lo"], case["hi"], case["seqs"]), _spread(case["n_lo"], case["n_hi"], case["seqs"])[::-1]))


def _parents(n, span):
    """A tree of n drafted tokens: the parent of token i is one of the `span` before it, or none (-1)."""
    return [i - 1 - (7 * i + i * i // 3) % min(i + 1, span) for i in range(n)]


def _seen(p, window, first):
    """How many of the positions 0 .. p a token at position p sees."""
    return p + 1 if not window or p < window else window + min(first, p + 1 - window)


def work(case):
    G, d, dv = case["G"], case["d"], case["dv"]
    row = d + dv + 8                         # codes and two scales of a token's head
    if case["op"] == "read":
        return {"bytes": case["rows"] * G * (row + (4 if case["out"] == "float32" else 2) * (d + dv)), "flops": case["rows"] * G * (d + dv)}
    lens = _lengths(case)
    T = sum(n for _, n in lens)
    if case["op"] == "write":
        return {"bytes": T * G * (row + (4 if case["x"] == "float32" else 2) * (d + dv)), "flops": 3 * T * G * (d + dv)}
    if case["op"] == "keep":
        moved = sum(min(case["path"], n) for _, n in lens)
        return {"bytes": 2 * moved * case["layers"] * G * row, "flops": 0}
    H, w, f = case["H"], case["window"], case["first"]
    pairs = rows = 0
    for past, n in lens:
        if case["op"] == "attn":
            # sum over the portion of what each token sees
            a, b = past, past + n - 1        # first and last position
            full = lambda p: (p + 1) * (p + 2) // 2  # noqa: E731
            if not w or b < w:
                pairs += full(b) - (full(a - 1) if a else 0)
            else:
                pairs += sum(_seen(p, w, f) for p in range(a, b + 1))
            low = max(0, a - w + 1) if w else 0
            rows += past + n - low + min(f, low)
        else:
            depth = []
            for i, p in enumerate(_parents(n, case["span"])):
                depth.append(depth[p] + 1 if p >= 0 else 0)
            pairs += sum(_seen(past + x, w, f) for x in depth)
            low = max(0, past - w + 1) if w else 0
            rows += past + n - low + min(f, low)
    qb, ob = (4 if case["q"] == "float32" else 2), (4 if case["out"] == "float32" else 2)
    return {"bytes": rows * G * row + T * H * (d * qb + dv * ob), "flops": 2 * pairs * H * (d + dv)}


# ------------------------------------------------------------------------------------------------ inputs

class Draws:
    """Tensors from the seed alone, on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 62))

    def n(self, *shape):
        return torch.randn(*shape, device=DEV, generator=self.g)

    def order(self, n):
        return torch.randperm(n, device=DEV, generator=self.g)


def _quantised(x, fmt):
    """(codes, scales) of fp32 rows x [..., n]; the quotients of the int8 form in 64 bits, as some of them lie next to a border."""
    a = x.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(x).all(-1, keepdim=True)
    if fmt == "e4m3":
        m, e = torch.frexp(a)
        k = torch.clamp(e - 9 + (m > 0.875).int(), min=-126)
        s = torch.where(a > 0, torch.ldexp(torch.ones_like(a), k), torch.zeros_like(a))
        c = (x / torch.where(s > 0, s, torch.ones_like(s))).nan_to_num(0.0, 0.0, 0.0).to(torch.float8_e4m3fn)
    else:
        s = a / 127.0
        t = torch.where(s > 0, s, torch.ones_like(s)).double()
        c = torch.round(x.double() / t).nan_to_num(0.0, 0.0, 0.0).clamp(-127, 127).to(torch.int8)
    c = torch.where(ok, c.view(torch.uint8), torch.zeros_like(c, dtype=torch.uint8)).view(c.dtype)
    return c, torch.where(ok, s, torch.full_like(s, float("nan"))).squeeze(-1)


def _pool(dr, pages, G, width, fmt, spread):
    """Pages full of rows as a model leaves them: normal numbers, rows of different sizes, some channels larger than others."""
    codes, scales = [], []
    channel = torch.exp(0.5 * dr.n(G, 1, width))
    for at in range(0, pages, 2048):
        n = min(2048, pages - at)
        x = dr.n(n, G, PAGE, width) * channel * torch.exp(spread * dr.n(n, G, PAGE, 1))
        c, s = _quantised(x, fmt)
        codes.append(c)
        scales.append(s)
    return torch.cat([c.view(torch.uint8) for c in codes]).view(CODE[fmt]), torch.cat(scales)


def prepare(case, seed):
    dr, fmt, G, d, dv = Draws(seed), case["fmt"], case["G"], case["d"], case["dv"]
    lens = [(case["first"], case["rows"])] if case["op"] == "read" else _lengths(case)
    layers = case.get("layers", 1)
    held = [(past + n + PAGE - 1) // PAGE for past, n in lens]
    total = sum(held) + 3
    order = dr.order(total).tolist()
    lists, at = [], 0
    for h in held:
        lists.append(order[at:at + h])
        at += h
    st = {"case": dict(case), "lens": lens, "scale": d ** -0.5}
    k, ks = _pool(dr, layers * total, G, d, fmt, 0.1)
    v, vs = _pool(dr, layers * total, G, dv, fmt, 0.3)
    st["k"], st["ks"], st["v"], st["vs"] = (t.view(layers, total, *t.shape[1:]) for t in (k, ks, v, vs))
    T = sum(n for _, n in lens)
    spans = [_parents(n, case["span"]) if "span" in case else [i - 1 for i in range(n)] for _, n in lens]
    if case["op"] in ("tree", "keep"):
        # the step's drafted tokens: row base + i holds token i, whose position is base + its depth
        st["parents"] = spans
    if case["op"] == "write":
        H = case["H"]
        proj = dr.n(T, H * d + G * d + G * dv) * torch.exp(0.3 * dr.n(T, 1))        # one projection [q | k | v]: rows far apart
        proj = proj.to(BF) if case["x"] == "bfloat16" else proj
        st["x_k"], st["x_v"] = proj[:, H * d:(H + G) * d].view(T, G, d), proj[:, (H + G) * d:].view(T, G, dv)
    if "q" in case:
        q = dr.n(T, case["H"], d)
        st["q"] = q.to(BF) if case["q"] == "bfloat16" else q
    if case["op"] == "keep":
        # an accepted path: rising numbers of drafted tokens, -1 behind its end
        P = case["path"]
        score = torch.rand(len(lens), max(n for _, n in lens), device=DEV, generator=dr.g)
        number = torch.arange(score.shape[1], device=DEV)
        n_of = torch.tensor([n for _, n in lens], device=DEV)[:, None]
        score = torch.where(number < n_of, score, torch.full_like(score, -1.0))
        top = torch.topk(score, min(P, score.shape[1]), dim=1)
        path = torch.where(top.values >= 0, top.indices, torch.full_like(top.indices, 1 << 20)).sort(1).values
        path = torch.where(path < 1 << 20, path, torch.full_like(path, -1))
        st["path"] = torch.cat([path, torch.full((len(lens), P - path.shape[1]), -1, device=DEV, dtype=path.dtype)], 1).to(torch.int32)
    if own:
        # what a serving program keeps: the cache, and the tables of the step that all layers share
        from krasis_b200 import seqops
        from krasis_b200.attention import CompactKVCache
        cache = CompactKVCache(layers, G, d, dv, DEV, max_pages=total, fmt=fmt, page_size=PAGE)
        cache.k.copy_(st.pop("k"))
        cache.v.copy_(st.pop("v"))
        cache.k_scale.copy_(st.pop("ks"))
        cache.v_scale.copy_(st.pop("vs"))
        st["cache"] = cache
        entries = [([0] * n, past, i, pages) for i, ((past, n), pages) in enumerate(zip(lens, lists))]
        if "parents" in st:
            st["tables"] = seqops.DraftTables([e + (p,) for e, p in zip(entries, spans)], DEV)
        else:
            st["tables"] = seqops.StepTables(entries, DEV)
        return st
    # the same as index tensors
    width = max(held)
    st["pages"] = torch.tensor([p + [0] * (width - len(p)) for p in lists], device=DEV)
    st["seq"] = torch.tensor([i for i, (_, n) in enumerate(lens) for _ in range(n)], device=DEV)
    st["row"] = torch.tensor([past + i for past, n in lens for i in range(n)], device=DEV)
    st["own_row"] = torch.tensor([i for _, n in lens for i in range(n)], device=DEV)
    st["base"], st["n"] = (torch.tensor([x[j] for x in lens], device=DEV) for j in (0, 1))
    N = max(n for _, n in lens)
    if "q" in case:
        depth, seen = [], torch.zeros(len(lens), N, N, dtype=torch.bool)
        for s, parents in enumerate(spans if case["op"] == "tree" else []):
            for i, p in enumerate(parents):
                depth.append(depth[len(depth) - i + p] + 1 if p >= 0 else 0)
                if p >= 0:
                    seen[s, i] = seen[s, p]
                seen[s, i, i] = True
        st["depth"] = torch.tensor(depth, device=DEV) if depth else None
        st["seen"] = seen.to(DEV)
    return st


# ------------------------------------------------------------------------------------------------ the plain forms

def _write(st):
    fmt, rows = st["case"]["fmt"], st["row"]
    page = st["pages"][st["seq"], rows // PAGE]
    for x, codes, scales in ((st["x_k"], st["k"], st["ks"]), (st["x_v"], st["v"], st["vs"])):
        c, s = _quantised(x.float(), fmt)
        codes[0].view(torch.uint8)[page, :, rows % PAGE] = c.view(torch.uint8)
        scales[0][page, :, rows % PAGE] = s
    return {"k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}


def _read(st):
    case = st["case"]
    rows = torch.arange(case["first"], case["first"] + case["rows"], device=DEV)
    page = st["pages"][0, rows // PAGE]
    dtype = BF if case["out"] == "bfloat16" else torch.float32
    back = lambda c, s: (c[0].view(torch.uint8)[page, :, rows % PAGE].view(c.dtype).float() * s[0][page, :, rows % PAGE][..., None]).to(dtype)  # noqa: E731
    return {"k": back(st["k"], st["ks"]), "v": back(st["v"], st["vs"])}


def _attend(st):
    """softmax(scale q k^T) v over whole page lists, what a token does not see masked."""
    case = st["case"]
    S, (H, G), (d, dv) = case["seqs"], (case["H"], case["G"]), (case["d"], case["dv"])
    R, N, L = H // G, st["seen"].shape[1], st["pages"].shape[1] * PAGE
    whole = lambda c, s, n: (c[0].view(torch.uint8)[st["pages"]].view(c.dtype).float() * s[0][st["pages"]][..., None]).transpose(1, 2).reshape(S, G, L, n)  # noqa: E731
    k, v = whole(st["k"], st["ks"], d), whole(st["v"], st["vs"], dv)
    q = torch.zeros(S, N, H, d, device=DEV)
    q[st["seq"], st["own_row"]] = st["q"].float()
    q = q.view(S, N, G, R, d).permute(0, 2, 1, 3, 4).reshape(S, G, N * R, d)
    scores = (q @ k.transpose(2, 3) * st["scale"]).view(S, G, N, R, L)
    j = torch.arange(L, device=DEV)
    at = torch.zeros(S, N, dtype=torch.int64, device=DEV)
    base = st["base"][:, None, None]
    if case["op"] == "tree":
        at[st["seq"], st["own_row"]] = st["base"][st["seq"]] + st["depth"]
        i = (j - base).expand(S, N, L)
        inside = (i >= 0) & (i < st["n"][:, None, None])
        i = i.clamp(0, N - 1)
        see = torch.where(inside, torch.gather(st["seen"], 2, i), j < base)
        spot = torch.where(inside, torch.gather(at[:, None].expand(S, N, N), 2, i), j)      # a key's position
    else:
        at[st["seq"], st["own_row"]] = st["row"]
        see, spot = j <= at[..., None], j
    if case["window"]:
        see = see & ((at[..., None] - spot < case["window"]) | (spot < case["first"]))
    scores = scores.masked_fill(~see[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    o = (p.view(S, G, N * R, L) @ v).view(S, G, N, R, dv) / p.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(S, N, H, dv)[st["seq"], st["own_row"]]
    return o.to(BF if case["out"] == "bfloat16" else torch.float32)


def _keep(st):
    path = st["path"].long()
    good = path >= 0
    seq = torch.arange(path.shape[0], device=DEV)[:, None].expand_as(path)[good]
    to = (st["base"][:, None] + torch.arange(path.shape[1], device=DEV))[good]
    frm = (st["base"][:, None] + path)[good]
    page_to, page_from = st["pages"][seq, to // PAGE], st["pages"][seq, frm // PAGE]
    for t in (st["k"].view(torch.uint8), st["v"].view(torch.uint8), st["ks"], st["vs"]):
        t[:, page_to, :, to % PAGE] = t[:, page_from, :, frm % PAGE]
    return {"k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}


def _own(st):
    from krasis_b200 import seqops
    case, cache, tb = st["case"], st["cache"], st["tables"]
    held = {"k": cache.k, "v": cache.v, "ks": cache.k_scale, "vs": cache.v_scale}
    if case["op"] == "write":
        seqops.kv_write(st["x_k"], st["x_v"], tb, cache, 0)
        return held
    if case["op"] == "keep":
        seqops.kv_keep(tb, st["path"], cache)
        return held
    dtype = BF if case["out"] == "bfloat16" else torch.float32
    if case["op"] == "read":
        k, v = seqops.kv_read(tb, 0, case["first"], case["rows"], cache, 0, dtype=dtype)
        return {"k": k, "v": v}
    call = seqops.kv_tree_attn if case["op"] == "tree" else seqops.kv_attn
    return call(st["q"], tb, cache, 0, st["scale"], window=case["window"] or None, first=case["first"], dtype=dtype)


def run(state):
    if own:
        return _own(state)
    return {"write": _write, "read": _read, "attn": _attend, "tree": _attend, "keep": _keep}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ 64 bits

def _back64(codes, scales):
    return codes.double() * scales.double()[..., None]


def _codes64(x, fmt):
    """Codes and scales of one tensor of rows [T, G, n] from the definition: the scale is held in fp32, the code is the nearest one to the exact quotient."""
    x = x.double()
    a = x.abs().amax(-1)
    if fmt == "int8":
        s = (a / 127).float()
        t = torch.where(s > 0, s, torch.ones_like(s)).double()[..., None]
        c = torch.round(x / t).clamp(-127, 127).to(torch.int8)
        return c, s
    k = torch.ceil(torch.log2(torch.where(a > 0, a, torch.ones_like(a)) / 448))
    k = torch.where(torch.exp2(k - 1) * 448 >= a, k - 1, torch.where(torch.exp2(k) * 448 < a, k + 1, k)).clamp(min=-126)
    s = torch.where(a > 0, torch.exp2(k), torch.zeros_like(a))
    y = x / torch.where(s > 0, s, torch.ones_like(s))[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)            # three bits behind the leading one, 2^-9 the least
    return (torch.round(y / step) * step).to(torch.float8_e4m3fn), s.float()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op, lens, pages = case["op"], st["lens"], st["pages"]
    if op == "keep":
        return None                          # rows are moved, nothing is computed
    if op == "write":
        for x, codes, scales in ((st["x_k"], st["k"], st["ks"]), (st["x_v"], st["v"], st["vs"])):
            c, s = _codes64(x, case["fmt"])
            flat = torch.arange(st["seq"].numel(), device=DEV)
            page, off = pages[st["seq"], st["row"] // PAGE], st["row"] % PAGE
            codes.view(torch.uint8)[0, page, :, off] = c.view(torch.uint8)[flat]
            scales[0, page, :, off] = s
        return {"k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}
    rows64 = lambda s, g, end, c, sc: _back64(c[0].view(torch.uint8)[pages[s], g].view(c.dtype), sc[0][pages[s], g]).reshape(-1, c.shape[-1])[:end]  # noqa: E731
    if op == "read":
        lo, hi = case["first"], case["first"] + case["rows"]
        both = [torch.stack([rows64(0, g, hi, c, sc)[lo:] for g in range(case["G"])], 1) for c, sc in ((st["k"], st["ks"]), (st["v"], st["vs"]))]
        return {"k": both[0], "v": both[1]}
    H, G, w = case["H"], case["G"], case["window"]
    R, T = H // G, sum(n for _, n in lens)
    o, at = torch.empty(T, H, case["dv"], dtype=torch.float64, device=DEV), 0
    for s, (past, n) in enumerate(lens):
        j = torch.arange(past + n, device=DEV)
        if op == "tree":
            p = past + st["depth"][at:at + n]
            see = torch.cat([torch.ones(n, past, dtype=torch.bool, device=DEV), st["seen"][s, :n, :n]], 1)
            spot = torch.cat([j[:past], p])
        else:
            p, spot = j[past:], j
            see = j[None] <= p[:, None]
        if w:
            see = see & ((p[:, None] - spot[None] < w) | (spot[None] < case["first"]))
        hide = ~see.repeat_interleave(R, 0)
        for g in range(G):
            k, v = rows64(s, g, past + n, st["k"], st["ks"]), rows64(s, g, past + n, st["v"], st["vs"])
            q = st["q"][at:at + n, g * R:(g + 1) * R].double().reshape(n * R, -1)
            z = (q @ k.T * st["scale"]).masked_fill_(hide, float("-inf"))
            z = torch.softmax(z, 1)
            o[at:at + n, g * R:(g + 1) * R] = (z @ v).view(n, R, -1)
        at += n
    return o
