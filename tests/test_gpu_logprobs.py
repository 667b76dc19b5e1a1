"""Log probabilities of given tokens, entropy and largest alternatives against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check(z, tokens, top):
    from krasis_b200 import seqops
    r = seqops.token_logprobs(z, tokens, top)
    T, V = z.shape
    assert r.logprob.shape == (T,) and r.entropy.shape == (T,) and r.top_ids.shape == (T, top) and r.top_logprobs.shape == (T, top) and r.top_ids.dtype is torch.int32
    if T == 0:
        return r
    z64 = z.double()
    bad = ~(z64 < float("inf")).all(1) | (z64 == -float("inf")).all(1)
    assert bool(r.logprob[bad].isnan().all()) and bool(r.entropy[bad].isnan().all()) and bool((r.top_ids[bad] == -1).all()) and bool(r.top_logprobs[bad].isnan().all())
    ok = ~bad
    if not bool(ok.any()):
        return r
    lp = torch.log_softmax(z64[ok], 1)
    inside = (tokens[ok] >= 0) & (tokens[ok] < V)
    want = torch.where(inside, lp.gather(1, tokens[ok].long().clamp(0, V - 1)[:, None])[:, 0], torch.full_like(lp[:, 0], -float("inf")))
    _near(r.logprob[ok], want, V)
    p = lp.exp()
    told = torch.where(p > 0, p * lp, torch.zeros_like(lp))
    # d = z - max is one rounding of d, so the sum of p d is off by 2^-24 |p d|, and by the weights' own error below
    size = (torch.where(p > 0, p * (z64[ok] - z64[ok].amax(1, keepdim=True)).abs(), torch.zeros_like(lp))).sum(1)
    off = _lse_off(V) * 2 * (1 + size) + 2.0 ** -23 * (size + told.sum(1).abs())
    assert bool(((r.entropy[ok].double() + told.sum(1)).abs() <= off).all())
    if top:
        ids = torch.sort(z[ok].float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids[ok].long(), ids)
        _near(r.top_logprobs[ok], lp.gather(1, ids), V)
    return r


def _lse_off(V):
    """How far the logarithm of the sum may be off: weights by exp to 2^-21 (two units in the last place of exp, one rounding of the argument, which is at most 104 where the
    weight is not lost: 104 2^-24 < 2^-17), sums of V terms by threads of 2^-24 each in at most 32 + V / 128 steps."""
    return 2.0 ** -17 + (32 + V / 128) * 2.0 ** -24


def _near(got, want, V):
    fin = torch.isfinite(want)
    assert torch.equal(got.double()[~fin], want[~fin])
    off = _lse_off(V) + 2.0 ** -22 * want[fin].abs()
    assert bool(((got.double()[fin] - want[fin]).abs() <= off).all()), float(((got.double()[fin] - want[fin]).abs() - off).max())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 7, 7), (3, 64, 64), (2, 257, 5), (4, 1000, 20), (1, 32768, 1), (4, 151936, 20), (5, 50001, 64), (33, 4099, 0), (300, 3001, 3), (700, 129, 2),
                                     (160, 40007, 8), (0, 100, 2)])
def test_rows(T, V, top, dtype):
    z = (torch.randn(T, V, device="cuda", generator=_gen(1)) * 3).to(dtype)
    tokens = torch.randint(0, V, (T,), device="cuda", generator=_gen(2))
    _check(z, tokens, top)
    _check(z, tokens.to(torch.int32), 0)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("pad", [1, 3, 8, 64])
def test_strides_and_odd_starts(dtype, pad):
    """Rows of a wider tensor, from any number on."""
    z = (torch.randn(6, 5000 + pad, device="cuda", generator=_gen(3)) * 2).to(dtype)
    tokens = torch.randint(0, 4990, (6,), device="cuda", generator=_gen(4))
    for first in (0, 1, pad):
        _check(z[:, first:first + 4993], tokens, 9)
    _check(z[::2, :4096], tokens[:3], 4)
    _check(z[:1].expand(4, -1), tokens[:4], 2)                                   # one row for all


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T", [3, 200])
def test_masked_and_equal_logits(T, dtype):
    """-inf weighs nothing; of equal logits the lowest id comes first; fewer numbers than alternatives; one number that is all; tokens outside; nothing but -inf, NaN, +inf."""
    V, inf = 6007, float("inf")
    z = (torch.randn(T, V, device="cuda", generator=_gen(5))).to(dtype)
    tokens = torch.randint(0, V, (T,), device="cuda", generator=_gen(6))
    z[0] = -inf
    z[0, 1234] = 2.0
    tokens[0] = 1234
    z[1] = 0.0
    z[1, ::2] = -0.0
    z[2, 100:] = -inf
    tokens[2] = 500
    _check(z, tokens, 64)
    tokens[0], tokens[1], tokens[2] = -1, V, 2 ** 40
    r = _check(z, tokens, 3)
    assert bool((r.logprob[:3] == -inf).all())
    z[0] = -inf
    z[1, 77] = float("nan")
    z[2, V - 1] = inf
    _check(z, tokens, 10)


@pytest.mark.parametrize("T,V", [(2, 151936), (150, 20000)])
@pytest.mark.parametrize("order", ["rising", "falling", "one block", "far apart", "few values"])
def test_orders(T, V, order):
    """Rows that pass every bound late, early or in one place, of numbers near and far, many of them equal."""
    i = torch.arange(V, device="cuda", dtype=F32)
    z = {"rising": i * 1e-3, "falling": -i * 1e-3, "one block": torch.where((i > 5000) & (i < 5300), i * 0.01, -i), "far apart": torch.sin(i * 12.9898) * 3e4,
         "few values": torch.floor(torch.sin(i * 78.233) * 3)}[order].repeat(T, 1)
    z += torch.arange(T, device="cuda")[:, None]
    _check(z, torch.arange(T, device="cuda") * 31 % V, 32)
    _check(z.to(BF), torch.arange(T, device="cuda") * 31 % V, 64)


@pytest.mark.parametrize("T", [2, 300])
def test_replayed_and_on_two_streams(T):
    from krasis_b200 import graphs, seqops
    z, tokens = torch.randn(T, 30011, device="cuda", generator=_gen(7)), torch.randint(0, 30011, (T,), device="cuda", generator=_gen(8))
    call = lambda: seqops.token_logprobs(z, tokens, 12)          # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [call() for _ in range(8)]
    here = [call() for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in other + here for a, b in zip(first, r))
    graph, out = graphs.capture(call, torch.device("cuda", 0))
    z.copy_(torch.randn(T, 30011, device="cuda", generator=_gen(9)))
    graph.replay()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, call()))
    _check(z, tokens, 12)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,V", [(1, 1500), (3, 1000), (2, 151936), (200, 4099), (400, 20000)])
def test_a_token_that_has_nearly_all_of_the_weight(T, V, dtype):
    """Its log probability is -log(1 + s) with s what the others weigh beside it: each weight is off by 2^-21 for the exponential and 2^-23 |d| for d = z - max and its product with
    log2 e, with |d| < 64 here 2^-17 in all, and the sum of positive numbers by 2^-24 for each of at most 32 + V / 128 steps; the logarithm and the last rounding 2^-22."""
    from krasis_b200 import seqops
    g = torch.Generator(device="cuda").manual_seed(T + V)
    z = torch.randn(T, V, device="cuda", generator=g) * 2
    tokens = torch.randint(0, V, (T,), device="cuda", generator=g)
    z[torch.arange(T), tokens] = 24.0 + 10 * torch.rand(T, device="cuda", generator=g)
    z = z.to(dtype)
    r = seqops.token_logprobs(z, tokens, 2)
    d = z.double() - z.double().amax(1, keepdim=True)
    d.scatter_(1, tokens[:, None], -float("inf"))
    want = -torch.log1p(d.exp().sum(1))
    off = 2.0 ** -17 + (32 + V / 128) * 2.0 ** -24 + 2.0 ** -22
    assert bool(((r.logprob.double() - want).abs() <= off * want.abs()).all()) and torch.equal(r.top_logprobs[:, 0], r.logprob)
