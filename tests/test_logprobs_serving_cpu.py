"""Scoring and log probabilities of the scheduler with a stand-in model on the CPU, where the operator is replaced by its definition."""
import json
import math

import pytest
import torch

from tests.test_serving_cpu import FakeModel


def _defined(z, tokens, top=0):
    from krasis_b200.seqops import TokenLogprobs
    lp = torch.log_softmax(z.double(), 1)
    best = lp.topk(top, 1) if top else None
    empty = lp.new_zeros(len(lp), 0)
    return TokenLogprobs(lp.gather(1, tokens[:, None].long())[:, 0], torch.special.entr(lp.exp()).sum(1), best.indices.int() if top else empty.int(), best.values if top else empty)


@pytest.fixture
def sched(monkeypatch):
    from krasis_b200 import seqops
    from krasis_b200.scheduler import Scheduler
    monkeypatch.setattr(seqops, "token_logprobs", _defined)
    return Scheduler(FakeModel(), max_tokens=64, max_requests=3)


def _logits(token, position):
    return -(torch.arange(13) - (token + position) % 13).abs().double()


@pytest.mark.parametrize("portion", [1, 2, 5, 100])
def test_scores(sched, portion):
    texts = [[1, 2, 3, 4, 5, 6, 7], [3], [], [2, 2]]
    got = sched.score(texts, step_tokens=portion)
    assert [len(g) for g in got] == [6, 0, 0, 1] and not sched.live and sched.kv_cache.free_page_count == 16
    for text, g in zip(texts, got):
        for i, s in enumerate(g):
            assert math.isclose(s, float(torch.log_softmax(_logits(text[i], i), 0)[text[i + 1]]), rel_tol=1e-9)


def test_generated_tokens_with_their_log_probabilities(sched):
    prompts = [[1, 2, 3], [4], [5, 6, 7, 8, 9]]
    ids = sched.generate(prompts, max_new_tokens=4, step_tokens=4)
    same, details = sched.generate(prompts, max_new_tokens=4, step_tokens=4, logprobs=3)
    assert same == ids and [len(d) for d in details] == [4, 4, 4]
    for p, out, told in zip(prompts, ids, details):
        seq = list(p)
        for tok, d in zip(out, told):
            lp = torch.log_softmax(_logits(seq[-1], len(seq) - 1), 0)
            assert math.isclose(d["logprob"], float(lp[tok]), rel_tol=1e-9) and len(d["top"]) == 3 and d["top"][0][0] == tok
            assert math.isclose(d["entropy"], float(torch.special.entr(lp.exp()).sum()), rel_tol=1e-9)
            seq.append(tok)
    assert sched.generate([], 2, logprobs=0) == ([], [])


def test_a_text_that_does_not_fit(sched):
    with pytest.raises(RuntimeError, match="does not fit"):
        sched.score([list(range(65))])
    with pytest.raises(ValueError):
        sched.score([[1, 2]], step_tokens=0)
    for bad in (-1, 65):
        with pytest.raises(ValueError):
            sched.generate([[1, 2]], 2, logprobs=bad)
    assert not sched.live and sched.kv_cache.free_page_count == 16


def test_more_alternatives_than_tokens(sched):
    ids, details = sched.generate([[1, 2, 3]], max_new_tokens=2, logprobs=64)
    assert len(ids[0]) == 2 and all(sorted(t for t, _ in d["top"]) == list(range(13)) for d in details[0]) and not sched.live


def test_perplexity():
    from krasis_b200.__main__ import perplexity
    assert perplexity([]) is None and perplexity([0.0, 0.0]) == 1 and math.isclose(perplexity([-1.0, -3.0]), math.exp(2))
    assert perplexity([-2e6, -1.0]) == perplexity([-math.inf]) == math.inf and math.isnan(perplexity([math.nan, -1.0]))


def test_designs_that_do_not_hold_their_experts_in_8_bits(tmp_path, capsys):
    from krasis_b200.__main__ import main
    for cfg in ({"architecture": "Kivurax"}, {"model_type": "qwen3_moe"}):
        (tmp_path / "config.json").write_text(json.dumps(cfg))
        assert main(["score", "--model", str(tmp_path), "--prompt-ids", "1,2", "--expert-format", "e4m3"]) == 3
        assert "does not hold its experts" in capsys.readouterr().err
