"""Log probabilities of logits up to the ends of their type."""
import pytest
import torch

from tests.test_gpu_logprobs import _check, _gen

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,V", [(4, 1000), (4, 70001), (300, 3001)])
def test_logits_near_the_largest_number(T, V, dtype):
    """Only a NaN or an infinity makes a row worthless: numbers up to the type's largest have the log probabilities that their differences give."""
    z = torch.randn(T, V, device="cuda", generator=_gen(11)).to(dtype)
    tokens = torch.randint(0, V, (T,), device="cuda", generator=_gen(12))
    big = torch.finfo(dtype).max
    z[0, V - 1] = z[0, 17] = big                                             # two that share all of the weight
    tokens[0] = 17
    z[1, 5] = 2.5e38
    tokens[1] = 5
    z[2] = 3e38                                                              # equal ones: log V each
    tokens[2] = V // 2
    z[3, 1:] = -big                                                          # one that is not masked
    tokens[3] = 0
    r = _check(z, tokens, 3)
    assert bool(torch.isfinite(r.logprob).all())
    lp = torch.log(torch.tensor([2.0, 1.0, V, 1.0], dtype=torch.float64))
    assert bool(((r.logprob[:4].double().cpu() + lp).abs() <= 2.0 ** -17 + 2.0 ** -20 * lp).all())


def test_differences_beyond_the_largest_number():
    """A log probability below the least fp32 number is -inf, and its row keeps the others."""
    from krasis_b200 import seqops
    z = torch.zeros(2, 500, device="cuda")
    z[:, 3], z[:, 4] = 3e38, -3e38
    r = seqops.token_logprobs(z, torch.tensor([4, 3], device="cuda"), 2)
    assert r.logprob.tolist() == [-float("inf"), 0.0] and r.entropy.tolist() == [0.0, 0.0] and r.top_ids.tolist() == [[3, 0]] * 2
    assert r.top_logprobs[:, 0].tolist() == [0.0, 0.0]
