"""Routed experts in 8 bits round once: a bfloat16 result is the fp32 one, rounded."""
import pytest
import torch

from tests import fp8_plain as plain
from tests.test_gpu_fp8 import _choices, _near, _rows, _weight, waits  # noqa: F401

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("T,top,E,W,F", [(1, 1, 1, 128, 128), (4, 10, 512, 512, 128), (9, 6, 16, 1040, 384), (130, 3, 5, 2048, 512), (333, 6, 64, 512, 256), (700, 8, 12, 400, 256)])
def test_a_bf16_result_is_the_fp32_one_rounded(T, top, E, W, F):
    from krasis_b200 import layers
    h = _rows(T, W, BF, 41)
    (w1, s1), (w2, s2) = _weight(E, 2 * F, W, 42), _weight(E, W, F, 43)
    ids, wt = _choices(T, top, E, 44)
    wt[:, top // 2] *= -1                                                    # sums that cancel
    ids[0, 0] = -1
    got, exact = (layers.fp8_experts(h, ids, wt, w1, s1, w2, s2, out_dtype=t) for t in (BF, F32))
    assert got.dtype is BF and exact.dtype is F32
    assert torch.equal(got, exact.to(BF))
    # what the fp32 one may be off by, and one rounding of half a step, 2^-8 of the result
    want, off = plain.experts(h, ids, wt, w1, s1, w2, s2, F32)
    _near(got, want, off + 2.0 ** -8 * (want.abs() + off))
