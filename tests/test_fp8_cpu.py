"""What the 8-bit floating-point operators and the log probabilities refuse, ahead of the device; and the plain implementation that they are tested against."""
import pytest
import torch

from tests import fp8_plain as plain

F8, BF = torch.float8_e4m3fn, torch.bfloat16


def _w(n, k, e=None):
    shape = (n, k) if e is None else (e, n, k)
    return torch.zeros(shape, dtype=F8), torch.ones(shape[:-2] + (plain.blocks(n), plain.blocks(k)))


def test_refusals_of_rows_and_blocks():
    from krasis_b200 import layers
    with pytest.raises(ValueError, match="one CUDA device"):
        layers.quantize_fp8_rows(torch.zeros(2, 32))
    for bad in (torch.zeros(2, 30), torch.zeros(32), torch.zeros(2, 0), torch.zeros(32, 64)[:, ::2], torch.zeros(16, 32).t()):
        with pytest.raises(ValueError):
            layers.quantize_fp8_rows(bad)
    with pytest.raises(ValueError, match="float16"):
        layers.quantize_fp8_rows(torch.zeros(2, 32, dtype=torch.float16))
    for bad in (torch.zeros(2, 30), torch.zeros(32), torch.zeros(0, 32), torch.zeros(32, 64).t(), torch.zeros(1, 2, 3, 16)):
        with pytest.raises(ValueError):
            layers.quantize_fp8_blocks(bad)
    with pytest.raises(ValueError, match="one CUDA device"):
        layers.quantize_fp8_blocks(torch.zeros(2, 32))


def test_refusals_of_products():
    from krasis_b200 import layers
    x, (w, s) = torch.zeros(2, 272), _w(300, 272)
    with pytest.raises(ValueError, match="one CUDA device"):
        layers.fp8_linear(x, w, s)
    for args in ((x, w.float(), s), (x, w[:, :256], s), (x, w, s[:2]), (x, w, s.t().contiguous()), (x, w, s.double()), (x[:, :256], w, s), (x, w.t().contiguous().t(), s)):
        with pytest.raises(ValueError):
            layers.fp8_linear(*args)
    for bias in (torch.zeros(299), torch.zeros(300, dtype=BF)):
        with pytest.raises(ValueError):
            layers.fp8_linear(x, w, s, bias=bias)
    c = torch.zeros(2, 272, dtype=F8)
    for args in ((x, torch.ones(2, 3)), (c, torch.ones(2, 2)), (c, torch.ones(3, 2).t().double()), (c.expand(2, 272)[:, :256], torch.ones(2, 2))):
        with pytest.raises(ValueError):
            layers.fp8_linear_rows(*args, w, s)


def test_refusals_of_experts():
    from krasis_b200 import layers
    h, ids, wt, (w1, s1), (w2, s2) = torch.zeros(5, 272), torch.zeros(5, 2, dtype=torch.int32), torch.zeros(5, 2), _w(256, 272, 3), _w(272, 128, 3)
    with pytest.raises(ValueError, match="one CUDA device"):
        layers.fp8_experts(h, ids, wt, w1, s1, w2, s2)
    for args in ((h, ids.long(), wt, w1, s1, w2, s2), (h, ids[:4], wt, w1, s1, w2, s2), (h, ids, wt[:, :1], w1, s1, w2, s2), (h, ids, wt.double(), w1, s1, w2, s2),
                 (h[:, :256], ids, wt, w1, s1, w2, s2), (h, ids, wt, w1[:, :200], s1, w2, s2), (h, ids, wt, w1, s1, w2[:2], s2[:2]), (h, ids, wt, w1, s1[:, :1], w2, s2),
                 (h, ids[:, :0], wt[:, :0], w1, s1, w2, s2), (h.half(), ids, wt, w1, s1, w2, s2)):
        with pytest.raises(ValueError):
            layers.fp8_experts(*args)


def test_refusals_of_the_c_interface(lib):
    """Sizes and workspaces are checked ahead of the device; nothing here reaches one."""
    from krasis_b200 import capi
    p = 1 << 20                                     # an address on 16 bytes that nobody reads
    bad = capi.KB2_ERR_VALUE
    assert lib.kb2_fp8_quantize_rows(p, 0, 32, 4, 24, p, p, 4, 0, None) == bad
    assert lib.kb2_fp8_quantize_rows(p, 0, 32, 4, 32, p + 8, p, 4, 0, None) == bad
    assert lib.kb2_fp8_quantize_rows(p, 0, 32, 4, 32, p, p, 3, 0, None) == bad
    assert lib.kb2_fp8_quantize_rows(p, 0, 32, -1, 32, p, p, 4, 0, None) == bad
    assert lib.kb2_fp8_quantize_rows(None, 0, 32, 0, 32, None, None, 0, 0, None) == capi.KB2_OK
    assert lib.kb2_fp8_quantize_blocks(p, 0, 1, 0, 32, p, p, 0, None) == bad
    assert lib.kb2_fp8_quantize_blocks(p, 0, 65536, 1, 32, p, p, 0, None) == bad
    assert lib.kb2_fp8_linear_rows(p, p, 4, p, p, None, p + 2, 0, 4, 16, 32, 0, None) == bad
    assert lib.kb2_fp8_linear_rows(p, p, 6, p, p, None, p, 0, 4, 16, 32, 0, None) == bad
    assert lib.kb2_fp8_linear_rows(p, p, 4, p, p, None, p, 0, 4, 0, 32, 0, None) == bad
    need = lib.kb2_fp8_linear_workspace(5, 48)
    assert need == 240 + 8 * 4
    assert lib.kb2_fp8_linear(p, 0, 48, p, p, None, p, 0, 5, 16, 48, p, need - 1, 0, None) == bad
    assert lib.kb2_fp8_linear(p, 0, 48, p, p, None, p, 0, 5, 16, 48, None, need, 0, None) == bad
    assert lib.kb2_fp8_experts_workspace(0, 2, 4, 128, 128, 0) == 0
    for sizes in ((4, 2, 1025, 128, 128), (4, 0, 4, 128, 128), (4, 2, 4, 120, 128), (4, 2, 4, 128, 64), (2 ** 30, 8, 4, 128, 128)):
        assert lib.kb2_fp8_experts_workspace(*sizes, 0) == 0
        assert lib.kb2_fp8_experts(p, 0, 128, p, p, p, p, p, p, p, 0, *sizes, p, 2 ** 40, 0, None) == bad
    need = lib.kb2_fp8_experts_workspace(4, 2, 4, 128, 128, 0)
    assert need > 0 and lib.kb2_fp8_experts(p, 0, 128, p, p, p, p, p, p, p, 0, 4, 2, 4, 128, 128, p, need - 1, 0, None) == bad
    assert lib.kb2_fp8_experts(p, 0, 128, p, None, p, p, p, p, p, 0, 4, 2, 4, 128, 128, p, need, 0, None) == bad


def test_refusals_of_log_probabilities():
    from krasis_b200 import seqops
    z, t = torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        seqops.token_logprobs(z, t)
    lib, p = seqops.load(), 1 << 20
    for args in ((p, 2, 50, 3, 50, p, 0), (p, 0, 50, -1, 50, p, 0), (p, 0, 50, 3, 0, p, 0), (p, 0, 50, 3, 50, p, 51), (p, 0, 500, 3, 500, p, 65), (p, 0, 50, 3, 50, p, -1), (p, 0, -1, 3, 50, p, 0),
                 (None, 0, 50, 3, 50, p, 0), (p, 0, 50, 3, 50, None, 0)):
        assert lib.kb2_seq_token_logprobs(*args, p, p, p, p, 0, None) == 2
    assert lib.kb2_seq_token_logprobs(p, 0, 50, 3, 50, p, 2, p, p, None, p, 0, None) == 2
    assert lib.kb2_seq_token_logprobs(None, 0, 50, 0, 50, None, 0, None, None, None, None, 0, None) == 0


def test_the_plain_quantisation():
    """Every e4m3 number is its own code, and the numbers next to the middle between two of them fall to either side."""
    codes = torch.arange(256, dtype=torch.uint8).view(F8).double()
    codes = codes[torch.isfinite(codes)]
    assert torch.equal(plain.nearest(codes), codes)
    pos = torch.sort(codes[codes >= 0].unique()).values
    mid = (pos[1:] + pos[:-1]) / 2
    assert torch.equal(plain.nearest(mid * (1 - 1e-9)), pos[:-1]) and torch.equal(plain.nearest(mid * (1 + 1e-9)), pos[1:])
    assert torch.equal(plain.nearest(mid), mid.float().to(F8).double())
    a = torch.tensor([0.0, 448.0, 448.0001, 1.75, 1.7500001, 2.0 ** -140, 3e38], dtype=torch.float64)
    assert plain.scale_of(a).tolist() == [0.0, 1.0, 2.0, 2.0 ** -8, 2.0 ** -7, 2.0 ** -126, 2.0 ** 120]
    x = torch.randn(9, 200, generator=torch.Generator().manual_seed(1)).double()
    c, s = plain.quantize_rows(x)
    assert c.shape == x.shape and s.shape == (9, 2) and float(((c * plain.spread_rows(s, 200) - x).abs() / x.abs().clamp(min=0.02)).max()) <= 2.0 ** -4
