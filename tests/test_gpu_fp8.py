"""Products of 8-bit floating-point numbers with a scale per block of 128 against 64 bits: quantising rows and matrices, the product, routed experts."""
import pytest
import torch

from tests import fp8_plain as plain

pytestmark = pytest.mark.gpu
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(M, K, dtype, seed, pad=0):
    """Rows that are `pad` numbers apart, of sizes that differ by block."""
    g = _gen(seed)
    x = torch.randn(M, K + pad, device="cuda", generator=g) * torch.exp(2 * torch.randn(M, 1, device="cuda", generator=g))
    x *= torch.exp(0.7 * torch.randn(1, K + pad, device="cuda", generator=g))
    return x.to(dtype)[:, :K]


def _weight(E, N, K, seed):
    g = _gen(seed)
    codes = (torch.randn(E, N, K, device="cuda", generator=g) * 100).clamp(-448, 448).to(F8)
    return codes, torch.exp(torch.randn(E, plain.blocks(N), plain.blocks(K), device="cuda", generator=g)) * 1e-4


def _same(got, want):
    assert torch.equal(got.double().nan_to_num(123.0), want.nan_to_num(123.0))


def _near(got, want, off):
    assert got.shape == want.shape and bool(torch.isfinite(want).all())
    worse = (got.double() - want).abs() - off
    assert float(worse.max()) <= 0, f"off by {float(worse.max()):.3g} more than allowed"


@pytest.fixture(autouse=True)
def waits():
    yield
    from krasis_b200 import capi
    capi.check_waits()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,K,pad", [(1, 16, 0), (3, 128, 0), (5, 144, 8), (17, 2048, 0), (100, 2064, 3), (333, 1040, 1), (1000, 640, 16), (0, 256, 0)])
def test_rows(M, K, pad, dtype):
    from krasis_b200 import layers
    x = _rows(M, K, dtype, 1, pad)
    c, s = layers.quantize_fp8_rows(x)
    assert c.dtype is F8 and c.shape == (M, K) and s.shape == (M, plain.blocks(K))
    cw, sw = plain.quantize_rows(x.double())
    _same(c, cw)
    _same(s, sw)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_every_exponent(dtype):
    """Blocks of each size that the type has, zeros, numbers at and next to 448 scales, denormals, ties; numbers that are not finite."""
    from krasis_b200 import layers
    big = torch.finfo(dtype).max
    x = torch.zeros(300, 128)
    for i in range(256):
        x[i] = torch.linspace(-1, 1, 128) * (2.0 ** (i - 130) if i < 250 else 1.0)
    x[256:270] = torch.tensor([448, 449, 450, 447, 446, 224, 225, 896, 895, 897, 1.75, 1.76, 3.5, 14.0])[:, None] * torch.linspace(-1, 1, 128)
    x[271, 5], x[272, 127], x[273, 0] = float("nan"), float("inf"), -float("inf")
    x[274] = 1e-45
    x[275], x[276, 3] = big, -big
    x[277, 64:] = torch.arange(64).float() + 0.5                             # ties among the codes
    x[278] = -0.0
    x = x.to(dtype).cuda()
    c, s = layers.quantize_fp8_rows(x)
    cw, sw = plain.quantize_rows(x.double())
    _same(c, cw)
    _same(s, sw)
    assert bool(s[271:274].isnan().all()) and not bool(c[271:274].float().any())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(16, 16), (128, 128), (1, 144), (129, 272), (1000, 2064), (3, 256, 640), (2, 100, 48)])
def test_blocks(shape, dtype):
    from krasis_b200 import layers
    w = torch.randn(shape, device="cuda", generator=_gen(2)).to(dtype)
    w[..., :1, :16] *= 37.0
    c, s = layers.quantize_fp8_blocks(w)
    assert c.shape == w.shape and s.shape == shape[:-2] + (plain.blocks(shape[-2]), plain.blocks(shape[-1]))
    for e in range(shape[0] if len(shape) == 3 else 1):
        one = (lambda t: t[e]) if len(shape) == 3 else (lambda t: t)
        cw, sw = plain.quantize_blocks(one(w).double())
        _same(one(c), cw)
        _same(one(s), sw)


def test_blocks_that_hold_nothing_or_no_number():
    from krasis_b200 import layers
    w = torch.randn(300, 400, device="cuda", generator=_gen(3))
    w[:128, 128:256] = 0
    w[200, 300] = float("nan")
    w[299, 399] = float("inf")
    c, s = layers.quantize_fp8_blocks(w)
    cw, sw = plain.quantize_blocks(w.double())
    _same(c, cw)
    _same(s, sw)
    assert float(s[0, 1]) == 0 and bool(s[1, 2].isnan()) and bool(s[2, 3].isnan())


SIZES = [(1, 16, 16), (1, 128, 128), (2, 129, 144), (4, 1000, 2048), (7, 100, 4112), (15, 2048, 272), (16, 640, 1024), (17, 641, 1040), (33, 256, 512), (64, 2050, 2048), (65, 300, 7168),
         (100, 1, 640), (128, 512, 128), (200, 999, 1296), (255, 257, 2064), (256, 4096, 512), (300, 2560, 640), (513, 1536, 1040), (1000, 520, 2048), (2500, 384, 256)]


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, out):
    from krasis_b200 import layers
    dtype = BF if (M + N) % 2 else F32
    x, (w, s) = _rows(M, K, dtype, 4), _weight(1, N, K, 5)
    bias = torch.randn(N, device="cuda", generator=_gen(6)) if N % 3 else None
    got = layers.fp8_linear(x, w[0], s[0], bias=bias, out_dtype=out)
    assert got.dtype is out
    y, off = plain.product(plain.rows_back(*plain.quantize_rows(x.double())), plain.matrix_back(w[0], s[0]))
    if bias is not None:
        y = y + bias.double()
        off = off + 2.0 ** -24 * (y.abs() + off)
    _near(got, y, off + plain.half_step(out) * (y.abs() + off))
    c, xs = layers.quantize_fp8_rows(x)
    assert torch.equal(got, layers.fp8_linear_rows(c, xs, w[0], s[0], bias=bias, out_dtype=out))
    assert torch.equal(got, layers.fp8_linear_rows(c, xs.contiguous(), w[0], s[0], bias=bias, out_dtype=out))


@pytest.mark.parametrize("M", [3, 40, 400])
def test_product_with_numbers_that_are_not_finite(M):
    """A row with a NaN gives a row of NaN and touches no other; a weight's block scaled by NaN its columns; zeros and large scales stay what they are."""
    from krasis_b200 import layers
    x, (w, s) = _rows(M, 512, F32, 7), _weight(1, 300, 512, 8)
    x[1, 100] = float("nan")
    x[2, 300] = float("inf")
    x[0] = 0
    s[0, 0, 0], s[0, 1, 1] = 0.0, float("nan")
    got = layers.fp8_linear(x, w[0], s[0], out_dtype=F32)
    assert bool(got[1:3].isnan().all()) and bool(got[:, 128:256].isnan().all())
    keep = [i for i in range(M) if i not in (1, 2)]
    cols = list(range(128)) + list(range(256, 300))
    assert not bool(got[0][cols].any())
    y, off = plain.product(plain.rows_back(*plain.quantize_rows(x[keep].double())), plain.matrix_back(w[0], s[0])[cols])
    _near(got[keep][:, cols], y, off + plain.half_step(F32) * (y.abs() + off))


@pytest.mark.parametrize("M", [0, 1, 5, 20, 300, 700])
def test_rows_do_not_depend_on_what_lies_behind_them(M):
    """Nothing behind the last row is written, and rows of a wider tensor are taken by their stride."""
    from krasis_b200 import capi, layers
    K, N = 656, 500
    wide = _rows(M + 2, K, BF, 9, pad=24)
    w, s = _weight(1, N, K, 10)
    got = layers.fp8_linear(wide[:M], w[0], s[0])
    assert torch.equal(got, layers.fp8_linear(wide[:M].contiguous(), w[0], s[0]))
    if M:
        out = torch.full((M + 3, N), 7.0, dtype=BF, device="cuda")
        c, xs = layers.quantize_fp8_rows(wide[:M])
        capi.check(capi.load().kb2_fp8_linear_rows(c.data_ptr(), xs.data_ptr(), xs.stride(1), w.data_ptr(), s.data_ptr(), None, out.data_ptr(), 0, M, N, K, 0,
                                                   torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out[:M], got) and bool((out[M:] == 7).all())


def _choices(T, top, E, seed, spare=0):
    g = _gen(seed)
    z = torch.randn(T, E + spare, device="cuda", generator=g) + torch.randn(1, E + spare, device="cuda", generator=g)
    best = torch.topk(z, top, dim=1)
    return best.indices.to(torch.int32).contiguous(), torch.softmax(best.values, 1).contiguous()


EXPERTS = [(1, 1, 1, 128, 128), (1, 8, 64, 512, 256), (3, 2, 4, 272, 128), (4, 10, 512, 512, 128), (9, 6, 16, 1040, 384), (40, 4, 8, 640, 256), (100, 8, 300, 256, 128), (130, 3, 5, 2048, 512),
           (333, 6, 64, 512, 256), (700, 2, 3, 400, 640), (1000, 10, 128, 256, 128), (2000, 1, 2, 256, 128), (50, 20, 40, 128, 128), (600, 17, 1024, 256, 128), (129, 2, 2, 384, 256), (5000, 2, 300, 128, 128)]


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("T,top,E,W,F", EXPERTS)
def test_experts(T, top, E, W, F, out):
    from krasis_b200 import layers
    h = _rows(T, W, BF if T % 2 else F32, 11, pad=16)
    (w1, s1), (w2, s2) = _weight(E, 2 * F, W, 12), _weight(E, W, F, 13)
    ids, wt = _choices(T, top, E, 14)
    got = layers.fp8_experts(h, ids, wt, w1, s1, w2, s2, out_dtype=out)
    assert got.dtype is out
    want, off = plain.experts(h, ids, wt, w1, s1, w2, s2, out)
    _near(got, want, off)


@pytest.mark.parametrize("T", [4, 60, 900])
def test_experts_that_are_left_out_or_chosen_twice(T):
    """Ids outside the experts bring nothing, the same expert twice counts twice, one expert can have all rows and most none, weights may be zero or negative."""
    from krasis_b200 import layers
    E, W, F, top = 12, 272, 128, 5
    h = _rows(T, W, BF, 15)
    (w1, s1), (w2, s2) = _weight(E, 2 * F, W, 16), _weight(E, W, F, 17)
    ids, wt = _choices(T, top, E, 18)
    ids[:, 1] = 7
    ids[0] = -1
    ids[1, 2:], ids[2] = E, 7
    ids[3, :2] = torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    wt[:, 3] *= -1
    wt[2:, 4] = 0
    got = layers.fp8_experts(h, ids, wt, w1, s1, w2, s2)
    want, off = plain.experts(h, ids, wt, w1, s1, w2, s2, BF)
    _near(got, want, off)
    assert not bool(got[0].any())
    assert not bool(layers.fp8_experts(h, torch.full_like(ids, -1), wt, w1, s1, w2, s2).any())


def test_experts_without_tokens():
    from krasis_b200 import layers
    (w1, s1), (w2, s2) = _weight(3, 256, 128, 19), _weight(3, 128, 128, 20)
    got = layers.fp8_experts(torch.empty(0, 128, dtype=BF, device="cuda"), torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(0, 2, device="cuda"), w1, s1, w2, s2)
    assert got.shape == (0, 128)


def test_a_row_that_is_not_finite_stays_alone_among_the_experts():
    from krasis_b200 import layers
    (w1, s1), (w2, s2) = _weight(4, 256, 256, 21), _weight(4, 256, 128, 22)
    for T in (6, 300):
        h = _rows(T, 256, F32, 23)
        ids, wt = _choices(T, 2, 4, 24)
        clean = layers.fp8_experts(h, ids, wt, w1, s1, w2, s2)
        h[5, 200] = float("nan")
        got = layers.fp8_experts(h, ids, wt, w1, s1, w2, s2)
        assert bool(got[5].isnan().all())
        keep = [i for i in range(T) if i != 5]
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("T", [5, 600])
def test_replayed_and_on_two_streams(T):
    """Captured calls give the eager bits with other inputs in the same places; two calls on two streams do not meet; the same call twice gives the same bits."""
    from krasis_b200 import graphs, layers
    E, W, F, top, N = 16, 512, 256, 4, 700
    h = _rows(T, W, BF, 25)
    (w1, s1), (w2, s2), (wl, sl) = _weight(E, 2 * F, W, 26), _weight(E, W, F, 27), _weight(1, N, W, 28)
    ids, wt = _choices(T, top, E, 29)

    def both():
        y = layers.fp8_experts(h, ids, wt, w1, s1, w2, s2)
        return y, layers.fp8_linear(y, wl[0], sl[0], out_dtype=F32)
    first = both()
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [both() for _ in range(8)]
    here = [both() for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in other + here for a, b in zip(first, got))
    graph, out = graphs.capture(both, torch.device("cuda", 0))
    h.copy_(_rows(T, W, BF, 30))
    new_ids, new_wt = _choices(T, top, E, 31)
    ids.copy_(new_ids)
    wt.copy_(new_wt)
    graph.replay()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, both()))


def test_quantised_then_multiplied():
    """A matrix through quantize_fp8_blocks, rows through quantize_fp8_rows, and their product: the three agree on what codes and scales mean, and the quantisation
    costs what e4m3 does: half a step, 2^-4, of either number."""
    from krasis_b200 import layers
    x, w = torch.randn(70, 1040, device="cuda", generator=_gen(32)), torch.randn(300, 1040, device="cuda", generator=_gen(33))
    c, s = layers.quantize_fp8_blocks(w)
    got = layers.fp8_linear(x, c, s)
    # numbers below 2^-6 scales lie on a grid of 2^-9 scales; with 448 scales = twice the largest number at most that is 2^-18 of it
    far = lambda t: 2.0 ** -4 * t.abs().double() + 2.0 ** -17 * float(t.abs().max())          # noqa: E731
    off = x.abs().double() @ far(w).T + far(x) @ (w.abs().double() + far(w)).T
    _near(got, x.double() @ w.double().T, off * (1 + 2.0 ** -10))
