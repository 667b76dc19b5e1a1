"""What the command line prints and refuses, with a stand-in model on the CPU."""
import json
import math

import pytest
import torch

from tests.test_logprobs_serving_cpu import _defined
from tests.test_serving_cpu import FakeModel


class Certain(FakeModel):
    """All of the weight is on one token; from position 2 on no logit is a number."""

    def forward_step(self, tb, want_rows):
        z = super().forward_step(tb, want_rows)
        if z is not None:
            z = torch.where(z == 0, z, torch.full_like(z, -math.inf))
            z[tb.positions[want_rows] >= 2] = math.nan
        return z


@pytest.fixture
def run(monkeypatch, capsys):
    from krasis_b200 import registry, seqops
    from krasis_b200.__main__ import main
    monkeypatch.setattr(seqops, "token_logprobs", _defined)
    monkeypatch.setattr(registry, "load_model", lambda *a, **k: Certain())

    def lines(*args):
        assert main([*args, "--model", "-", "--max-tokens", "64"]) == 0
        not_json = lambda name: pytest.fail(f"{name} is not JSON")          # noqa: E731
        return [json.loads(line, parse_constant=not_json) for line in capsys.readouterr().out.splitlines()]
    return lines


def test_scores_are_json_whatever_the_numbers_are(run):
    """At position p the token after t is (t + p) % 13."""
    certain, cannot_be, no_number, nothing = run("score", "--prompt-ids", "5,5,6", "--prompt-ids", "5,7", "--prompt-ids", "5,5,6,8", "--prompt-ids", "3")
    assert certain == {"prompt_tokens": 3, "logprobs": [0.0, 0.0], "perplexity": 1.0}
    assert cannot_be == {"prompt_tokens": 2, "logprobs": [None], "perplexity": None}
    assert no_number == {"prompt_tokens": 4, "logprobs": [0.0, 0.0, None], "perplexity": None}
    assert nothing == {"prompt_tokens": 1, "logprobs": [], "perplexity": None}


def test_generated_tokens_are_json_whatever_the_numbers_are(run):
    (got,) = run("generate", "--prompt-ids", "5", "--max-new-tokens", "2", "--logprobs", "2")
    assert got["generated"][0] == 5 and len(got["logprobs"]) == 2
    assert got["logprobs"][0]["logprob"] == 0 and got["logprobs"][0]["top"][0] == [5, 0.0] and got["logprobs"][0]["top"][1][1] is None
    (got,) = run("generate", "--prompt-ids", "5,5,6", "--max-new-tokens", "1", "--logprobs", "1")
    assert got["logprobs"][0]["logprob"] is None and got["logprobs"][0]["entropy"] is None


@pytest.mark.parametrize("args,said", [(["generate", "--logprobs", "65"], "0 to 64"), (["generate", "--logprobs", "-1"], "0 to 64"), (["score", "--step-tokens", "0"], "at least one")])
def test_numbers_out_of_range_are_refused_ahead_of_loading(monkeypatch, capsys, args, said):
    from krasis_b200 import registry
    from krasis_b200.__main__ import main
    monkeypatch.setattr(registry, "load_model", lambda *a, **k: pytest.fail("loaded"))
    with pytest.raises(SystemExit) as e:
        main([*args, "--model", "-", "--prompt-ids", "1"])
    assert e.value.code == 2 and said in capsys.readouterr().err
