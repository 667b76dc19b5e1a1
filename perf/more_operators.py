"""Products of numbers held in 8-bit floating point with a scale for each block of 128, and the scoring of what a model answers, as cases that can be timed and checked.

  rows      rows of activations are quantised, a scale per 128 numbers of a row
  blocks    matrices of weights are quantised, a scale per block of 128 x 128
  linear    rows times a matrix that is held in 8 bits: quantises the rows, multiplies, adds a bias
  experts   routed experts whose matrices are held in 8 bits: sum over a token's choices of weight * down(silu(gate h) * up h)
  logprobs  log probabilities of given tokens, the entropy, and the largest alternatives of rows of logits

  own (set by whoever imports this)   False: elementary torch operations; True: the calls that a program makes of krasis_b200
  listed() / draw(rng)                the cases; prepare(case, seed) / run(state) one pass; work(case) what it cannot do without;
  exact(case, seed)                   the same from the definition in 64 bits

The format, per block with largest magnitude a: e4m3 codes, scale 2^k, the least k >= -126 with a <= 448 2^k; codes are the nearest ones to number / scale, ties to
even.  A matrix that comes with scales of its own (any fp32 numbers) is multiplied with those.
"""
import math

import torch

own = False

DEV = "cuda:0"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn
B = 128                                      # numbers a scale serves, along each axis


def listed():
    return [
        # one step of four decoded requests ahead of a product: latency
        {"name": "rows_step", "op": "rows", "M": 4, "K": 2048, "x": "bfloat16"},
        # a long prompt's rows, an odd number of them, ahead of a product of the largest preset's width
        {"name": "rows_prompt", "op": "rows", "M": 8191, "K": 4096, "x": "float32"},
        # one projection of a checkpoint in bfloat16 is brought into 8 bits, its last blocks cut
        {"name": "blocks_one", "op": "blocks", "E": 1, "N": 1000, "K": 2064, "x": "bfloat16"},
        # a layer's gate and up projections of all experts
        {"name": "blocks_experts", "op": "blocks", "E": 64, "N": 2816, "K": 2048, "x": "bfloat16"},
        # four requests decode through the widest projection of the flagship: the weights' way from memory
        {"name": "linear_step", "op": "linear", "M": 4, "N": 12288, "K": 2048, "x": "bfloat16", "out": "bfloat16", "bias": False},
        # a mixed step of prompt portions and decoded tokens, odd sizes, the result in fp32
        {"name": "linear_mixed", "op": "linear", "M": 333, "N": 4100, "K": 5136, "x": "float32", "out": "float32", "bias": True},
        # a prompt of 8192 tokens through the same projection: tensor cores
        {"name": "linear_prompt", "op": "linear", "M": 8192, "N": 12288, "K": 2048, "x": "bfloat16", "out": "bfloat16", "bias": False},
        # four requests decode through ten of 512 small experts each
        {"name": "experts_step", "op": "experts", "T": 4, "top": 10, "E": 512, "W": 2048, "F": 512, "x": "bfloat16"},
        # a mixed step through six of 64 larger experts, unevenly loaded
        {"name": "experts_mixed", "op": "experts", "T": 389, "top": 6, "E": 64, "W": 2048, "F": 1408, "x": "bfloat16"},
        # a prompt of 8192 tokens through ten of 512 experts: the flagship's layer
        {"name": "experts_prompt", "op": "experts", "T": 8192, "top": 10, "E": 512, "W": 2048, "F": 512, "x": "bfloat16"},
        # four decoded requests report their tokens' log probabilities with twenty alternatives
        {"name": "logprobs_step", "op": "logprobs", "T": 4, "V": 151936, "x": "float32", "top": 20},
        # a window of a text is scored: perplexity, no alternatives but the best
        {"name": "logprobs_text", "op": "logprobs", "T": 2048, "V": 151936, "x": "float32", "top": 1},
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rows", "blocks", "linear", "experts", "logprobs"])
    x = rng.choice(["bfloat16", "float32"])
    if op == "rows":
        return {"op": op, "M": _logint(rng, 1, 8192), "K": 16 * _logint(rng, 8, 512), "x": x}
    if op == "blocks":
        return {"op": op, "E": _logint(rng, 1, 16), "N": _logint(rng, 100, 4096), "K": 16 * _logint(rng, 8, 448), "x": x}
    if op == "linear":
        return {"op": op, "M": _logint(rng, 1, 8192), "N": _logint(rng, 100, 8192), "K": 16 * _logint(rng, 16, 360), "x": x,
                "out": rng.choice(["bfloat16", "float32"]), "bias": rng.choice([False, True])}
    if op == "experts":
        E = 2 ** rng.randint(3, 8)
        return {"op": op, "T": _logint(rng, 1, 4096), "top": rng.randint(1, 8), "E": E, "W": 16 * _logint(rng, 16, 192), "F": 128 * rng.randint(1, 8), "x": "bfloat16"}
    return {"op": op, "T": _logint(rng, 1, 2048), "V": _logint(rng, 1000, 140000), "x": x, "top": rng.randint(0, 32)}


def _wide(kind):
    return 4 if kind == "float32" else 2


def _blocks(n):
    return (n + B - 1) // B


def work(case):
    op = case["op"]
    if op == "rows":
        n, s = case["M"] * case["K"], case["M"] * _blocks(case["K"])
        return {"bytes": n * (_wide(case["x"]) + 1) + 4 * s, "flops": 3 * n}
    if op == "blocks":
        n, s = case["E"] * case["N"] * case["K"], case["E"] * _blocks(case["N"]) * _blocks(case["K"])
        return {"bytes": n * (_wide(case["x"]) + 1) + 4 * s, "flops": 3 * n}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K * _wide(case["x"]) + N * K + 4 * _blocks(N) * _blocks(K) + M * N * _wide(case["out"]) + (4 * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    if op == "experts":
        T, top, E, W, F = (case[k] for k in ("T", "top", "E", "W", "F"))
        met = E * (1.0 - (1.0 - top / E) ** T) if top < E else E          # experts that some token chose, about
        return {"bytes": int(T * W * 2 * _wide(case["x"]) + 8 * T * top + met * (3 * F * W + 12 * _blocks(F) * _blocks(W))), "flops": 6 * T * top * W * F}
    return {"bytes": case["T"] * (case["V"] * _wide(case["x"]) + 12 + 8 * case["top"]), "flops": 6 * case["T"] * case["V"]}


# ------------------------------------------------------------------------------------------------ inputs

class Draws:
    """Tensors from the seed alone, on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 62))

    def n(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=self.g, dtype=dtype)


def _weight(dr, E, N, K):
    """E matrices of a checkpoint that is held in 8 bits: codes, and scales that are any fp32 numbers."""
    codes = torch.empty(E, N, K, dtype=F8, device=DEV)
    at_once = max(1, (1 << 28) // (N * K))
    for e in range(0, E, at_once):
        n = min(at_once, E - e)
        codes[e:e + n] = dr.n(n, N, K, dtype=BF).mul_(100.0).clamp_(-448, 448).to(F8)
    return codes, torch.exp(0.3 * dr.n(E, _blocks(N), _blocks(K))) * (0.01 * K ** -0.5)


def _activations(dr, T, W, kind):
    """Rows as they leave a norm: some channels larger than others, a few numbers far out."""
    x = dr.n(T, W) * torch.exp(0.5 * dr.n(1, W))
    x = x * torch.where(dr.n(1, W) > 3.0, 20.0, 1.0)
    return x.to(BF) if kind == "bfloat16" else x


def prepare(case, seed):
    dr, op = Draws(seed), case["op"]
    st = {"case": dict(case)}
    if op == "rows":
        st["x"] = _activations(dr, case["M"], case["K"], case["x"])
    elif op == "blocks":
        st["w"] = torch.empty(case["E"], case["N"], case["K"], dtype=BF if case["x"] == "bfloat16" else torch.float32, device=DEV)
        for e in range(case["E"]):
            st["w"][e] = dr.n(case["N"], case["K"]) * 0.02
    elif op == "linear":
        st["x"] = _activations(dr, case["M"], case["K"], case["x"])
        w, s = _weight(dr, 1, case["N"], case["K"])
        st["w"], st["s"] = w[0], s[0]
        st["bias"] = dr.n(case["N"]) if case["bias"] else None
    elif op == "experts":
        T, top, E, W, F = (case[k] for k in ("T", "top", "E", "W", "F"))
        st["h"] = _activations(dr, T, W, case["x"])
        st["w1"], st["s1"] = _weight(dr, E, 2 * F, W)
        st["w2"], st["s2"] = _weight(dr, E, W, F)
        z = dr.n(T, E) + 0.5 * dr.n(1, E)                                  # some experts are liked more than others
        best = torch.topk(z, min(top, E), dim=1)
        st["ids"] = best.indices.to(torch.int32)
        st["weights"] = torch.softmax(best.values, 1)
    else:
        T, V = case["T"], case["V"]
        z = dr.n(T, V).mul_(2.0) + dr.n(1, V)
        st["tokens"] = torch.where(dr.n(T) > 0, torch.argmax(z, 1), torch.randint(0, V, (T,), device=DEV, generator=dr.g))
        z[:, V - V // 50:] = float("-inf")                                 # the padding of the vocabulary
        z[torch.arange(T, device=DEV), st["tokens"]] += 6.0
        st["z"] = z.to(BF) if case["x"] == "bfloat16" else z
    return st


# ------------------------------------------------------------------------------------------------ the plain forms

def _scale(a):
    """2^k, the least k >= -126 with a <= 448 2^k; 0 for a = 0."""
    m, e = torch.frexp(a)
    k = torch.clamp(e - 9 + (m > 0.875).int(), min=-126)
    return torch.where(a > 0, torch.ldexp(torch.ones_like(a), k), torch.zeros_like(a))


def _quantised_rows(x):
    """(codes [M, K], scales [M, blocks]) of fp32 rows."""
    M, K = x.shape
    p = torch.nn.functional.pad(x, (0, -K % B)).view(M, -1, B)
    s = _scale(p.abs().amax(-1))
    c = (p / torch.where(s > 0, s, torch.ones_like(s))[..., None]).to(F8)
    return c.view(M, -1)[:, :K].contiguous(), s


def _quantised_blocks(w):
    """(codes [N, K], scales [blocks, blocks]) of an fp32 matrix."""
    N, K = w.shape
    p = torch.nn.functional.pad(w, (0, -K % B, 0, -N % B)).view(_blocks(N), B, _blocks(K), B)
    s = _scale(p.abs().amax((1, 3)))
    c = (p / torch.where(s > 0, s, torch.ones_like(s))[:, None, :, None]).to(F8)
    return c.view(_blocks(N) * B, -1)[:N, :K].contiguous(), s


def _rows_back(c, s):
    return c.float() * s.repeat_interleave(B, 1)[:, :c.shape[1]]


def _matrix_back(c, s):
    return c.float() * s.repeat_interleave(B, 0)[:c.shape[0]].repeat_interleave(B, 1)[:, :c.shape[1]]


def _experts(st):
    h, ids, weights, (E, F2, W) = st["h"], st["ids"], st["weights"], st["w1"].shape
    F = F2 // 2
    x = _rows_back(*_quantised_rows(h.float()))
    y = torch.zeros(ids.shape[0], ids.shape[1], W, device=DEV)
    order = torch.argsort(ids.reshape(-1), stable=True)
    ends = torch.searchsorted(ids.reshape(-1)[order].contiguous(), torch.arange(E + 1, device=DEV, dtype=torch.int32)).tolist()
    for e in range(E):
        slots = order[ends[e]:ends[e + 1]]
        if slots.numel() == 0:
            continue
        gu = x[slots // ids.shape[1]] @ _matrix_back(st["w1"][e], st["s1"][e]).T
        g = gu[:, :F]
        a = _rows_back(*_quantised_rows(g / (1 + torch.exp(-g)) * gu[:, F:]))
        y.view(-1, W)[slots] = a @ _matrix_back(st["w2"][e], st["s2"][e]).T
    return (y * weights[..., None]).sum(1).to(h.dtype)


def _logprobs(st):
    z, top = st["z"].float(), st["case"]["top"]
    m = z.amax(1, keepdim=True)
    d = z - m
    p = torch.exp(d)
    total = p.sum(1, dtype=torch.float64).float()
    lse = torch.log(total)
    told = torch.where(p > 0, p * d, torch.zeros_like(p)).sum(1, dtype=torch.float64).float()
    out = {"logprob": d.gather(1, st["tokens"][:, None])[:, 0] - lse, "entropy": lse - told / total}
    if top:
        # the largest first, the lowest index among equals
        best = torch.sort(d, dim=1, descending=True, stable=True)
        out["ids"], out["best"] = best.indices[:, :top].to(torch.int32), best.values[:, :top] - lse[:, None]
    return out


def run(state):
    op = state["case"]["op"]
    out = {"bfloat16": BF, "float32": torch.float32}[state["case"].get("out", "bfloat16")]
    if own:
        from krasis_b200 import layers, seqops
        if op == "rows":
            c, s = layers.quantize_fp8_rows(state["x"])
            return {"codes": c, "scales": s}
        if op == "blocks":
            c, s = layers.quantize_fp8_blocks(state["w"])
            return {"codes": c, "scales": s}
        if op == "linear":
            return layers.fp8_linear(state["x"], state["w"], state["s"], bias=state["bias"], out_dtype=out)
        if op == "experts":
            return layers.fp8_experts(state["h"], state["ids"], state["weights"], state["w1"], state["s1"], state["w2"], state["s2"])
        r = seqops.token_logprobs(state["z"], state["tokens"], top=state["case"]["top"])
        got = {"logprob": r.logprob, "entropy": r.entropy}
        if state["case"]["top"]:
            got["ids"], got["best"] = r.top_ids, r.top_logprobs
        return got
    if op == "rows":
        c, s = _quantised_rows(state["x"].float())
        return {"codes": c, "scales": s}
    if op == "blocks":
        made = [_quantised_blocks(w.float()) for w in state["w"]]
        return {"codes": torch.stack([c.view(torch.uint8) for c, _ in made]).view(F8), "scales": torch.stack([s for _, s in made])}
    if op == "linear":
        y = _rows_back(*_quantised_rows(state["x"].float())) @ _matrix_back(state["w"], state["s"]).T
        return (y if state["bias"] is None else y + state["bias"]).to(out)
    return _experts(state) if op == "experts" else _logprobs(state)


# ------------------------------------------------------------------------------------------------ 64 bits

def _power(a):
    """The scale of a block whose largest magnitude is a, from the definition."""
    k = torch.ceil(torch.log2(torch.where(a > 0, a, torch.ones_like(a)) / 448))
    k = torch.where(torch.exp2(k - 1) * 448 >= a, k - 1, torch.where(torch.exp2(k) * 448 < a, k + 1, k)).clamp(min=-126)
    return torch.where(a > 0, torch.exp2(k), torch.zeros_like(a))


def _nearest(y):
    """The e4m3 number nearest to y, |y| <= 448, ties to even: three bits behind the leading one, 2^-9 the least step."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _row_codes(x):
    """Of rows [M, K] in 64 bits: (numbers that the codes stand for ahead of their scale, scales)."""
    M, K = x.shape
    c, s = torch.empty_like(x), torch.empty(M, _blocks(K), dtype=torch.float64, device=DEV)
    for b in range(_blocks(K)):
        part = x[:, b * B:(b + 1) * B]
        s[:, b] = _power(part.abs().amax(1))
        c[:, b * B:(b + 1) * B] = _nearest(part / torch.where(s[:, b] > 0, s[:, b], torch.ones_like(s[:, b]))[:, None])
    return c, s


def _whole(c, s):
    """A matrix from its codes and scales, in 64 bits."""
    w = c.double()
    for b in range(s.shape[1]):
        w[:, b * B:(b + 1) * B] *= s[:, b].double().repeat_interleave(B)[:w.shape[0], None]
    return w


def _whole_rows(c, s):
    x = c.clone()
    for b in range(s.shape[1]):
        x[:, b * B:(b + 1) * B] *= s[:, b:b + 1]
    return x


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "rows":
        c, s = _row_codes(st["x"].double())
        return {"codes": c, "scales": s}
    if op == "blocks":
        E, N, K = st["w"].shape
        codes = torch.empty(E, N, K, dtype=F8, device=DEV)
        scales = torch.empty(E, _blocks(N), _blocks(K), dtype=torch.float64, device=DEV)
        for e in range(E):
            w = st["w"][e].double()
            a = torch.stack([torch.stack([w[i * B:(i + 1) * B, j * B:(j + 1) * B].abs().max() for j in range(_blocks(K))]) for i in range(_blocks(N))])
            scales[e] = _power(a)
            one = torch.where(scales[e] > 0, scales[e], torch.ones_like(a))
            codes[e] = _nearest(w / one.repeat_interleave(B, 0)[:N].repeat_interleave(B, 1)[:, :K]).to(F8)
        return {"codes": codes, "scales": scales}
    if op == "linear":
        y = _whole_rows(*_row_codes(st["x"].double())) @ _whole(st["w"], st["s"]).T
        return y if st["bias"] is None else y + st["bias"].double()
    if op == "experts":
        ids, wt, (E, F2, W) = st["ids"].long(), st["weights"].double(), st["w1"].shape
        F = F2 // 2
        x = _whole_rows(*_row_codes(st["h"].double()))
        out = torch.zeros(ids.shape[0], W, dtype=torch.float64, device=DEV)
        for e in range(E):
            t, j = torch.nonzero(ids == e, as_tuple=True)
            if t.numel() == 0:
                continue
            z = x[t] @ _whole(st["w1"][e], st["s1"][e]).T
            a = _whole_rows(*_row_codes(z[:, :F] * torch.sigmoid(z[:, :F]) * z[:, F:]))
            out.index_add_(0, t, wt[t, j, None] * (a @ _whole(st["w2"][e], st["s2"][e]).T))
        return out
    z, tokens, top = st["z"], st["tokens"], case["top"]
    T = z.shape[0]
    logprob, entropy = (torch.empty(T, dtype=torch.float64, device=DEV) for _ in range(2))
    ids = torch.empty(T, top, dtype=torch.int32, device=DEV)
    best = torch.empty(T, top, dtype=torch.float64, device=DEV)
    for t in range(0, T, 64):
        lp = torch.log_softmax(z[t:t + 64].double(), 1)
        n = torch.arange(lp.shape[0], device=DEV)
        logprob[t:t + 64] = lp[n, tokens[t:t + 64]]
        entropy[t:t + 64] = torch.special.entr(lp.exp()).sum(1)
        if top:
            got = torch.sort(z[t:t + 64], dim=1, descending=True, stable=True).indices[:, :top]
            ids[t:t + 64], best[t:t + 64] = got.to(torch.int32), lp.gather(1, got)
    out = {"logprob": logprob, "entropy": entropy}
    if top:
        out["ids"], out["best"] = ids, best
    return out
