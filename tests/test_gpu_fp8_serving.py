"""8-bit floating-point experts and log probabilities where a user meets them: the routed-expert block, a model that is served, its text scores, and all of the operators one after the other."""
import json

import pytest
import torch

from tests import fp8_plain as plain

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rnd(*shape, seed, sd=1.0):
    return torch.randn(*shape, device="cuda", generator=_gen(seed)) * sd


def _block(E, W, F, shared, seed=1):
    w = {"router": _rnd(E, W, seed=seed, sd=0.3)}
    for e in range(E):
        w.update({f"e{e}_gate": _rnd(F, W, seed=10 + e, sd=0.1), f"e{e}_up": _rnd(F, W, seed=300 + e, sd=0.1), f"e{e}_down": _rnd(W, F, seed=600 + e, sd=0.1)})
    if shared:
        w.update({"shared_gate": _rnd(shared, W, seed=900, sd=0.1), "shared_up": _rnd(shared, W, seed=901, sd=0.1), "shared_down": _rnd(W, shared, seed=902, sd=0.1)})
    return {k: v.cpu() for k, v in w.items()}


@pytest.mark.parametrize("T", [1, 7, 90, 700])
@pytest.mark.parametrize("shared", [0, 48])
def test_a_block_of_experts_in_8_bits(T, shared):
    """RoutedExperts with expert_format "e4m3" against 64 bits, on the block's own choices and weights; the shared expert is as without it."""
    from krasis_b200.mixers import RoutedExperts
    E, W, F, top = 6, 272, 128, 2
    w = _block(E, W, F, shared)
    mod = RoutedExperts(w, E, 0, top, F32, "cuda:0", renorm=True, expert_format="e4m3")
    h = _rnd(T, W, seed=2)
    got = mod.forward(h)
    ids, wt, _ = mod.route(h)
    codes = lambda n: [plain.quantize_blocks(t.cuda().double()) for t in n]          # noqa: E731
    gu = codes([torch.cat([w[f"e{e}_gate"], w[f"e{e}_up"]]) for e in range(E)])
    down = codes([w[f"e{e}_down"] for e in range(E)])
    stack = lambda p, i: torch.stack([x[i] for x in p])                              # noqa: E731
    want, off = plain.experts(h, ids, wt, stack(gu, 0), stack(gu, 1), stack(down, 0), stack(down, 1), F32)
    if shared:
        side = mod.shared.forward(h).double()
        want = want + side
        off = off + 2.0 ** -23 * (want.abs() + side.abs() + off)
    worse = (got.double() - want).abs() - off
    assert float(worse.max()) <= 0, float(worse.max())


def test_what_a_block_of_experts_in_8_bits_refuses():
    from krasis_b200.mixers import RoutedExperts
    for kw, F, W in (({"act": "relu2", "gated": False}, 128, 32), ({"weight_input": True}, 128, 32), ({}, 96, 32), ({}, 128, 24)):
        with pytest.raises(ValueError):
            RoutedExperts(_block(2, W, F, 0), 2, 0, 1, F32, "cuda:0", expert_format="e4m3", **kw)
    w = _block(2, 32, 128, 0)
    w["router"] = torch.zeros(3, 32)
    with pytest.raises(ValueError):
        RoutedExperts(w, 2, 1, 1, F32, "cuda:0", expert_format="e4m3")
    with pytest.raises(ValueError):
        RoutedExperts(_block(2, 32, 128, 0), 2, 0, 1, F32, "cuda:0", expert_format="e5m2")


@pytest.mark.parametrize("T", [3, 200])
def test_all_of_them_in_a_row(T):
    """A checkpoint's matrices into 8 bits, experts on them, an 8-bit head, the log probabilities of what follows: each step against 64 bits on what the one before it gave."""
    from krasis_b200 import layers, seqops
    E, W, F, V, top = 8, 384, 128, 5000, 3
    gu, sgu = layers.quantize_fp8_blocks(_rnd(E, 2 * F, W, seed=3, sd=0.05).to(BF))
    dn, sdn = layers.quantize_fp8_blocks(_rnd(E, W, F, seed=4, sd=0.05).to(BF))
    head, shead = layers.quantize_fp8_blocks(_rnd(V, W, seed=5, sd=0.2).to(BF))
    h = _rnd(T, W, seed=6).to(BF)
    best = torch.topk(_rnd(T, E, seed=7), top, dim=1)
    ids, wt = best.indices.to(torch.int32), torch.softmax(best.values, 1)
    y = layers.fp8_experts(h, ids, wt, gu, sgu, dn, sdn)
    want, off = plain.experts(h, ids, wt, gu, sgu, dn, sdn, BF)
    assert bool(((y.double() - want).abs() <= off).all())
    z = layers.fp8_linear(y, head, shead, out_dtype=F32)
    want, off = plain.product(plain.rows_back(*plain.quantize_rows(y.double())), plain.matrix_back(head, shead))
    off = off + plain.half_step(F32) * (want.abs() + off)
    assert bool(((z.double() - want).abs() <= off).all())
    tokens = torch.randint(0, V, (T,), device="cuda", generator=_gen(8))
    r = seqops.token_logprobs(z, tokens, 5)
    lp = torch.log_softmax(z.double(), 1)
    assert float((r.logprob.double() - lp[torch.arange(T), tokens]).abs().max()) <= 2.0 ** -16
    assert torch.equal(r.top_ids.long(), torch.sort(z, dim=1, descending=True, stable=True).indices[:, :5])


def _model(fmt):
    from krasis_b200.megolorn import MegolornConfig, MegolornModel, random_weights
    from tests import test_gpu_megolorn as M
    mlp = M.moe(experts=5, identity=0, top=2, groups=1, keep=1, ff=128, shared=40)
    cfg = MegolornConfig.from_dict(M.model_cfg([M.L(M.attn_cfg(), M.dense()), M.L(M.attn_cfg(kv_from=0, chunk=5), mlp)]))
    model = MegolornModel(cfg, random_weights(cfg, 21), dtype=F32, expert_format=fmt)
    model.page_size = 4
    return model, M.toks


@pytest.mark.parametrize("fmt", [None, "e4m3"])
def test_a_served_model_scores_texts_and_tells_of_its_tokens(fmt):
    from krasis_b200.scheduler import Scheduler
    model, toks = _model(fmt)
    texts = [toks(n, 50, n) for n in (23, 1, 40)] + [[]]
    s = Scheduler(model, max_tokens=256, max_requests=3)
    for portion in (512, 16):
        got = s.score(texts, step_tokens=portion)
        assert [len(g) for g in got] == [22, 0, 39, 0] and not s.live
        for text, g in zip(texts, got):
            if len(text) < 2:
                continue
            z = [s.step([("t", text[a:a + portion], list(range(len(text[a:a + portion]))))]) for a in range(0, len(text), portion)]
            s.finish("t")
            lp = torch.log_softmax(torch.cat(z).double(), 1)[torch.arange(len(text) - 1), torch.tensor(text[1:])]
            assert float((torch.tensor(g, device="cuda").double() - lp).abs().max()) <= 2.0 ** -17 + 2.0 ** -22 * float(lp.abs().max())
    prompts = [toks(n, 50, 90 + n) for n in (9, 3, 17, 5)]
    plain_ids = s.generate(prompts, max_new_tokens=6, step_tokens=16)
    ids, details = s.generate(prompts, max_new_tokens=6, step_tokens=16, logprobs=4)
    assert ids == plain_ids and [len(d) for d in details] == [6] * 4
    for out, told in zip(ids, details):
        for tok, d in zip(out, told):
            assert d["top"][0] == (tok, d["logprob"]) and len(d["top"]) == 4          # greedy: the token is the most likely one
            assert 0 <= d["entropy"] <= 3.92 and all(a[1] >= b[1] for a, b in zip(d["top"], d["top"][1:]))          # log 50 = 3.912
    json.dumps(details)
