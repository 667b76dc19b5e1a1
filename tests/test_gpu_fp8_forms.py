"""Products of 8-bit floating-point numbers in the forms that small sizes do not take: two and four CTAs along K, pairs and single CTAs with several tiles each; experts whose rows are not on 16 bytes."""
import pytest
import torch

from tests import fp8_plain as plain
from tests.test_gpu_fp8 import _choices, _gen, _near, _rows, _weight, waits  # noqa: F401

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32

# by the form that 148 SMs give: tiles of 128 x 256 on single CTAs, of 256 x 256 on pairs
TWO, FOUR = [(4, 12288, 2048), (333, 4100, 5136)], [(129, 3000, 4112), (333, 2048, 4112)]
SINGLE = [(4096, 2560, 256), (4000, 2501, 400), (3000, 2564, 528)]                          # 320, 320 and 264 tiles
PAIRS = [(5000, 1024, 1024), (2500, 5000, 1296), (2500, 5004, 1296), (4900, 1030, 1168), (2300, 4999, 1168)]          # 80, 200, 200, 100 and 180 tiles of 74 pairs


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("M,N,K", TWO + FOUR + SINGLE + PAIRS)
def test_product(M, N, K, out):
    """Cut blocks of K, rows and columns; results on 16 bytes, on 8 and on neither; the same bits again and from rows that are quantised already."""
    from krasis_b200 import layers
    x, (w, s) = _rows(M, K, BF if N % 2 else F32, 51), _weight(1, N, K, 52)
    bias = torch.randn(N, device="cuda", generator=_gen(53)) if M % 2 == 0 else None
    got = layers.fp8_linear(x, w[0], s[0], bias=bias, out_dtype=out)
    y, off = plain.product(plain.rows_back(*plain.quantize_rows(x.double())), plain.matrix_back(w[0], s[0]))
    if bias is not None:
        y = y + bias.double()
        off = off + 2.0 ** -24 * (y.abs() + off)
    _near(got, y, off + plain.half_step(out) * (y.abs() + off))
    c, xs = layers.quantize_fp8_rows(x)
    for _ in range(3):
        assert torch.equal(got, layers.fp8_linear_rows(c, xs, w[0], s[0], bias=bias, out_dtype=out))


@pytest.mark.parametrize("M,N,K", [TWO[1], FOUR[0], SINGLE[1], PAIRS[3]])
def test_nothing_behind_the_last_row_is_written(M, N, K):
    from krasis_b200 import capi, layers
    (w, s), (c, xs) = _weight(1, N, K, 54), layers.quantize_fp8_rows(_rows(M, K, BF, 55))
    for dtype in (BF, F32):
        out = torch.full((M + 3, N), 7.0, dtype=dtype, device="cuda")
        capi.check(capi.load().kb2_fp8_linear_rows(c.data_ptr(), xs.data_ptr(), xs.stride(1), w.data_ptr(), s.data_ptr(), None, out.data_ptr(), int(dtype is F32), M, N, K, 0,
                                                   torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out[:M], layers.fp8_linear_rows(c, xs, w[0], s[0], out_dtype=dtype)) and bool((out[M:] == 7).all())


def test_rows_that_are_not_finite_stay_alone_among_tiles():
    """In the second tile of a pair as in the first."""
    from krasis_b200 import layers
    M, N, K = PAIRS[0]
    x, (w, s) = _rows(M, K, BF, 56), _weight(1, N, K, 57)
    clean = layers.fp8_linear(x, w[0], s[0])
    bad = [3, 300, 2559, 4999]
    x[bad, 500] = float("nan")
    got = layers.fp8_linear(x, w[0], s[0])
    assert bool(got[bad].isnan().all())
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[bad] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,top", [(1, 3), (60, 5), (1500, 3)])          # 4500 choices are placed in three launches
@pytest.mark.parametrize("pad,first", [(1, 0), (3, 0), (16, 1), (5, 3)])
def test_rows_of_experts_off_16_bytes(T, top, pad, first, dtype):
    """Rows of any stride, from any number on: the bits of the same rows side by side."""
    from krasis_b200 import layers
    E, W, F = 12, 272, 128
    h = _rows(T, W + first, dtype, 58, pad)[:, first:]
    assert h.data_ptr() % 16 or h.stride(0) % 8
    (w1, s1), (w2, s2) = _weight(E, 2 * F, W, 59), _weight(E, W, F, 60)
    ids, wt = _choices(T, top, E, 61)
    got = layers.fp8_experts(h, ids, wt, w1, s1, w2, s2)
    assert torch.equal(got, layers.fp8_experts(h.contiguous(), ids, wt, w1, s1, w2, s2))
    _near(got, *plain.experts(h, ids, wt, w1, s1, w2, s2, dtype))
