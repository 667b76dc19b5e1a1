"""Attention over the 8-bit cache in steps of portions, trees and decoded tokens side by side: partial results of the rows that are cut, and of no others."""
import pytest
import torch

from tests import kv_plain
from tests.test_gpu_kv_cache import BF, F32, _cache, _check, _gen, _step, _tree, forms, waits  # noqa: F401

pytestmark = pytest.mark.gpu

MIXED = {"cut and whole": [(1, 5000), (70, 900), (1, 40), (100, 3000), (1, 2500)], "whole first": [(40, 10), (1, 3), (1, 9000), (0, 64), (33, 6000)],
         "many short": [(1, 11 * i) for i in range(70)] + [(90, 4000), (1, 4000)], "all alike": [(24, 1500 * i) for i in range(4)], "long alone": [(3, 20000)]}


@pytest.mark.parametrize("H,G,d,dv", [(16, 2, 128, 128), (4, 4, 64, 64), (8, 2, 128, 256), (7, 7, 96, 80)])
@pytest.mark.parametrize("step", sorted(MIXED))
def test_mixed(H, G, d, dv, step, forms):  # noqa: F811
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step(MIXED[step], 64, 60)
    c = _cache(G, d, dv, pages, "int8", seed=61)
    q = torch.randn(tb.T, H, d, generator=_gen(62)).to(BF).cuda()
    for window, first in ((None, 0), (2000, 70)):
        known = None
        for do in (BF, F32):
            for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, d ** -0.5, window=window, first=first, dtype=do)):
                known = _check(got, q, c, seqs, known=known, scale=d ** -0.5, window=window, first=first)


def test_mixed_trees(forms):  # noqa: F811
    from krasis_b200 import seqops as ops
    lens = [(16, 5000), (64, 9000), (1, 700), (3, 8000), (40, 3)]
    tb, seqs, pages = _step(lens, 64, 63, parents=[_tree(n, n, 4) for n, _ in lens])
    c = _cache(2, 128, 128, pages, "e4m3", seed=64)
    q = torch.randn(tb.T, 16, 128, generator=_gen(65)).to(BF).cuda()
    for window, first in ((None, 0), (3000, 5)):
        known = None
        for got in forms(tb, lambda: ops.kv_tree_attn(q, tb, c, 0, 0.09, window=window, first=first)):
            known = _check(got, q, c, seqs, known=known, scale=0.09, window=window, first=first)


@pytest.mark.parametrize("decode,portion", [([30000], (4096, 0)), ([500 + 950 * i for i in range(32)], (2048, 5001))])
def test_a_portion_beside_long_requests(decode, portion):
    """The memory that a call takes beside its result, and the rows as a call of either kind alone gives them (bf16 results: a rounding apart, and the sums' order)."""
    from krasis_b200 import seqops as ops
    H, G, d = 64, 4, 128
    lens = [(1, n) for n in decode] + [portion]
    tb, seqs, pages = _step(lens, 64, 66)
    c = _cache(G, d, d, pages, "int8", seed=67)
    q = torch.randn(tb.T, H, d, generator=_gen(68)).to(BF).cuda()
    out = torch.empty(tb.T, H, d, dtype=BF, device="cuda")
    ops.kv_attn(q, tb, c, 0, 0.09, out=out)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.kv_attn(q, tb, c, 0, 0.09, out=out)
    assert torch.cuda.max_memory_allocated() - before <= len(decode) * H * 64 * 130 * 4 + (1 << 20)
    at = len(decode)
    for rows, part in ((slice(0, at), seqs[:-1]), (slice(at, None), seqs[-1:])):
        alone = ops.kv_attn(q[rows], ops.StepTables([([0] * n, s, 0, p) for n, s, p, _ in part], "cuda"), c, 0, 0.09)
        # either is within off_by of the truth; of a row's own largest number their parts come to 2^-7 of roundings and 2^-9 of weights and decoded numbers, for both
        far = (alone.float() - out[rows].float()).abs().amax(-1) / alone.float().abs().amax(-1)
        assert float(far.max()) <= 2.0 ** -6
    for i in {0, at // 5, at - 1}:
        _check(out[i:i + 1], q[i:i + 1], c, seqs[i:i + 1], scale=0.09)


def test_captured_mixed_steps(monkeypatch):
    """A captured step of a portion and decoded tokens, run again with other positions: cut by the room in the page lists."""
    from krasis_b200 import seqops as ops
    from krasis_b200.graphs import capture
    monkeypatch.setattr(ops, "KV_TILES_FROM", 17)
    H, G, d, ns, room = 8, 2, 128, (1, 40, 1, 9), 96
    c, g = _cache(G, d, d, 4 * room, "int8", 64, seed=69), _gen(70)
    pages = torch.randperm(4 * room, generator=g).tolist()
    lists, T = [pages[i * room:(i + 1) * room] for i in range(4)], sum(ns)
    q = torch.randn(T, H, d, generator=g).to(BF).cuda()
    buf = torch.zeros(3 * T + 5 + 4 + 4 * room, dtype=torch.int32, device="cuda")
    tables = lambda starts: ops.StepTables([([0] * n, s, i, lists[i]) for i, (n, s) in enumerate(zip(ns, starts))], "cuda", device_buf=buf)  # noqa: E731
    tb = tables((3, 40, 0, 7))
    graphs = [(w, do, capture(lambda w=w, do=do: ops.kv_attn(q, tb, c, 0, 0.09, window=w, first=3, dtype=do), "cuda")) for w, do in ((None, BF), (700, BF), (None, F32))]
    for starts in ((3, 40, 0, 7), (6143, 0, 5000, 6000), (0, 6104, 17, 3000), (0, 0, 0, 0)):
        kept = tables(starts)
        for _, _, (graph, _) in graphs:
            graph.replay()
        torch.cuda.synchronize()
        seqs = [(n, s, lists[i], None) for i, (n, s) in enumerate(zip(ns, starts))]
        for w, do, (_, out) in graphs:
            _check(out, q, c, seqs, scale=0.09, window=w, first=3)
        del kept


def test_steps_without_tokens():
    """Every call on a step that brings no tokens, and rows read back through such tables."""
    from krasis_b200 import seqops as ops
    c = _cache(2, 64, 32, 4, "int8", seed=71)
    entries = [([], 100, 0, [2, 0]), ([], 0, 1, [])]
    tb, dt = ops.StepTables(entries, "cuda"), ops.DraftTables([e + ([],) for e in entries], "cuda")
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    k, v, q = (torch.zeros(0, h, n, device="cuda") for h, n in ((2, 64), (2, 32), (4, 64)))
    for tables in (tb, dt):
        ops.kv_write(k, v, tables, c, 0)
    ops.kv_keep(dt, torch.zeros(2, 3, dtype=torch.int32, device="cuda"), c)
    for a, b in zip(before, (c.k, c.v, c.k_scale, c.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for do in (BF, F32):
        assert ops.kv_attn(q, tb, c, 0, 0.1, dtype=do).shape == ops.kv_tree_attn(q, dt, c, 0, 0.1, dtype=do).shape == (0, 4, 32)
    want = kv_plain.held(c, 0)
    for tables in (tb, dt):
        for got, x in zip(ops.kv_read(tables, 0, 60, 40, c, 0, dtype=F32), want):
            rows = x[[2, 0]].transpose(1, 2).reshape(-1, 2, x.shape[-1])[60:100]
            assert bool(((got.double().cpu() - rows).abs() <= rows.abs() * 2.0 ** -24).all())
        with pytest.raises(IndexError):
            ops.kv_read(tables, 1, 0, 1, c, 0)


def test_a_workspace_that_is_too_small_is_refused():
    """With a buffer of the size that is needed, of which one byte less is declared."""
    import ctypes as C

    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 5000), (70, 900)], 64, 72)
    c = _cache(2, 128, 128, pages, "int8", seed=73)
    q, out = torch.randn(tb.T, 16, 128, generator=_gen(74)).cuda(), torch.full((tb.T, 16, 128), 7.0, device="cuda")
    lib, st = ops.load(), ops._kv_step(tb)[0]
    size = lib.kb2_seq_kv_attn_workspace(c.address, st, 16, 0, 0, 0)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    call = lambda n: lib.kb2_seq_kv_attn(c.address, 0, st, q.data_ptr(), 0, 16 * 128, 128, 16, C.c_float(0.09), 0, 0, None, out.data_ptr(), 0, work.data_ptr(), n,  # noqa: E731
                                         torch.cuda.current_stream().cuda_stream)
    assert size > 0 and call(size - 1) == 2 and bool((out == 7).all())
    assert call(size) == 0
    _check(out, q, c, seqs, scale=0.09)
