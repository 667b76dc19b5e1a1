"""Holding a checkpoint's experts in 8 bits takes what the codes take."""
import pytest
import torch

from tests import fp8_plain as plain
from tests.test_gpu_fp8_serving import _block

pytestmark = pytest.mark.gpu


def test_memory_while_experts_are_brought_into_8_bits():
    """At its peak: the codes and scales, and of one matrix the fp32 numbers, a copy of them and its codes."""
    from krasis_b200.mixers import RoutedExperts
    E, W, F = 64, 512, 256
    w = _block(E, W, F, 0)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    mod = RoutedExperts(w, E, 0, 2, torch.bfloat16, "cuda:0", expert_format="e4m3")
    torch.cuda.synchronize()
    codes = 3 * E * W * F
    assert mod.w_gu.numel() + mod.w_down.numel() == codes
    assert torch.cuda.max_memory_allocated() - before <= codes * (1 + 4 / 128 ** 2) + 2 * F * W * (2 * 4 + 1) + 2 ** 20
    for e in (0, E - 1):
        for got, s, want in ((mod.w_gu[e], mod.s_gu[e], torch.cat([w[f"e{e}_gate"], w[f"e{e}_up"]])), (mod.w_down[e], mod.s_down[e], w[f"e{e}_down"])):
            c, scale = plain.quantize_blocks(want.cuda().double())
            assert torch.equal(got.double(), c) and torch.equal(s.double(), scale)
