"""Attention over the 8-bit cache where rows of values are zero or far apart, and where a step's tables hold fewer tokens than its layout."""
import pytest
import torch

from tests import kv_plain
from tests.test_gpu_kv_cache import BF, F32, _cache, _check, _gen, _step, _tree, forms, waits  # noqa: F401

pytestmark = pytest.mark.gpu


def _zero(c, seqs, rows):
    """Zero values in the rows that `rows` says of every sequence."""
    for n, start, pages, _ in seqs:
        for j in rows(start + n):
            c.v[0, pages[j // c.page_size], :, j % c.page_size] = 0
            c.v_scale[0, pages[j // c.page_size], :, j % c.page_size] = 0


GROUPS = {"first": lambda n: range(min(n, 16)), "of the first warps": lambda n: [j for j in range(n) if j < 128 and j // 16 % 3],
          "of all warps": lambda n: range(min(n, 128)), "of each piece": lambda n: [j for j in range(n) if j // 16 % 16 < 9], "every other": lambda n: [j for j in range(n) if j // 16 % 2 == 0],
          "the first row": lambda n: [0], "all but the last": lambda n: range(n - 1)}


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("H,G,d,dv", [(16, 2, 128, 128), (4, 4, 64, 64), (6, 2, 256, 256)])
@pytest.mark.parametrize("groups", sorted(GROUPS))
def test_rows_of_zero_values(fmt, H, G, d, dv, groups, forms):  # noqa: F811
    """Rows whose values are all zero weigh in the sum and take nothing from the rows behind them."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 500), (1, 20), (30, 300), (1, 3000)], 64, 40)
    c = _cache(G, d, dv, pages, fmt, seed=41)
    _zero(c, seqs, GROUPS[groups])
    q = torch.randn(tb.T, H, d, generator=_gen(42)).cuda()
    for window, first in ((None, 0), (200, 1), (40, 16)):
        known = None
        for do in (F32, BF):
            for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, d ** -0.5, window=window, first=first, dtype=do)):
                known = _check(got, q, c, seqs, known=known, scale=d ** -0.5, window=window, first=first)


@pytest.mark.parametrize("groups", ["first", "of all warps", "every other"])
def test_rows_of_zero_values_ahead_of_drafts(groups, forms):  # noqa: F811
    from krasis_b200 import seqops as ops
    lens = [(16, 5000), (40, 64), (3, 300)]
    tb, seqs, pages = _step(lens, 64, 43, parents=[_tree(n, n, 4) for n, _ in lens])
    c = _cache(2, 128, 128, pages, "int8", seed=44)
    _zero(c, seqs, GROUPS[groups])
    q = torch.randn(tb.T, 16, 128, generator=_gen(45)).cuda()
    known = None
    for do in (F32, BF):
        for got in forms(tb, lambda: ops.kv_tree_attn(q, tb, c, 0, 0.09, dtype=do)):
            known = _check(got, q, c, seqs, known=known, scale=0.09)


def test_many_keys_behind_rows_of_zero_values():
    """Keys that are cut evenly over the GPU, and a captured-size step of few keys that clusters join."""
    from krasis_b200 import seqops as ops
    for lens, H, G, d in (([(1, 20000 + 97 * i) for i in range(3)], 12, 12, 128), ([(2, 7000)] * 5, 16, 4, 256), ([(1, 900)] * 4, 16, 2, 128)):
        tb, seqs, pages = _step(lens, 64, 46)
        c = _cache(G, d, d, pages, "int8", seed=47)
        _zero(c, seqs, lambda n: [j for j in range(n) if j // 16 % 32 < 20])
        q = torch.randn(tb.T, H, d, generator=_gen(48)).cuda()
        known = None
        for do in (F32, BF):
            known = _check(ops.kv_attn(q, tb, c, 0, d ** -0.5, dtype=do), q, c, seqs, known=known, scale=d ** -0.5)
@pytest.mark.parametrize("H,G,d,dv", [(16, 2, 128, 128), (4, 4, 64, 64), (6, 2, 256, 256)])
@pytest.mark.parametrize("above", [60.0, 83.0, 84.5, 85.5, 86.5, 90.0])
def test_a_zero_value_far_above_large_ones(H, G, d, dv, above, forms):  # noqa: F811
    """One key takes nearly all of the weight and its value is zero, as are those around it: the others' large values count for next to nothing, and for a number."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 700), (40, 900)], 64, 49)
    c = _cache(G, d, dv, pages, "int8", seed=50)
    c.k.copy_(torch.randint(-3, 4, c.k.shape, generator=_gen(51), dtype=torch.int8))
    c.k_scale.fill_(1.0)
    c.v_scale[0].copy_(torch.exp2(torch.randint(13, 17, c.v_scale[0].shape, generator=_gen(52)).float()))
    c.v_scale[0, :, :, ::7] *= 2.0 ** 20
    _zero(c, seqs, lambda n: range(256, 400))
    for n, start, pl, _ in seqs:
        c.k[0, pl[300 // 64], :, 300 % 64] = 100
    q = torch.ones(tb.T, H, d).cuda()
    scale = above / (100 * d)
    want, *sizes = kv_plain.attention(q, c, 0, seqs, scale)
    # Beside off_by.  Weights are fp32 numbers relative to the row's largest, and the exponential gives 0 below 2^-126: each is off by as much, and the result by that times
    # the sum of |v|.  A reference is at least 2^-100 of the unit that it divides (on tiles), and a product is off by half of fp16's least step, 2^-25, times it: 2^-125 of |v|.
    # Products of weight and unit up to 1e-37 may be left out, the unit at least 2^-7 of the row's scale: 1e-37 times 2^7 times the sum of the codes.
    numbers, codes = kv_plain.held(c, 0)[1].abs(), c.v[0].cpu().double().abs()
    lost, at = torch.zeros_like(want), 0
    for n, start, pl, _ in seqs:
        for x, f in ((numbers, 3 * 2.0 ** -126), (codes, 2.0 ** 7 * 1e-37)):
            lost[at:at + n] += f * x[pl].transpose(1, 2).reshape(-1, G, dv)[:start + n].sum(0).repeat_interleave(H // G, 0)
        at += n
    for do in (F32, BF):
        off = kv_plain.off_by(F32, do, 940, d, want, *sizes, decoded=True) + lost
        for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, scale, dtype=do)):
            assert bool(torch.isfinite(got).all())
            err = (got.double().cpu() - want).abs()
            assert bool((err <= off).all()), (float((err / off).max()), float(err.max()))


@pytest.mark.parametrize("lens,keep,tiles_from", [([(1, 300), (30, 200), (12, 100)], 39, 40), ([(20, 500)], 3, 17), ([(1, 900), (1, 20), (50, 700), (13, 0), (40, 31)], 66, 33),
                                                  ([(12, 700)] * 3, 26, 48), ([(64, 2000), (64, 3000)], 70, 0), ([(1, 4000), (12, 3000), (20, 0)], 5, 24)])
@pytest.mark.parametrize("H,G,d", [(8, 2, 128), (8, 2, 256)])
@pytest.mark.parametrize("tree", [False, True])
def test_fewer_tokens_than_the_layout_has(lens, keep, tiles_from, H, G, d, tree, monkeypatch):
    """The device's table of first tokens ends early: what is left of a sequence that was planned for the tiles has few rows, and is attended to all the same."""
    from krasis_b200 import seqops as ops
    monkeypatch.setattr(ops, "KV_TILES_FROM", tiles_from)
    tb, seqs, pages = _step(lens, 64, 53, parents=[_tree(n, n, 4) for n, _ in lens] if tree else None)
    c = _cache(G, d, d, pages, "int8", seed=54)
    T, at = tb.T, 0
    tb.cu.clamp_(max=keep)
    for i, (n, start, pl, parents) in enumerate(seqs):
        left = max(0, min(n, keep - at))
        at += n
        seqs[i] = (left, start, pl, parents[:left] if tree else None)
    q = torch.randn(T, H, d, generator=_gen(55)).to(BF).cuda()
    call = ops.kv_tree_attn if tree else ops.kv_attn
    for window, first in ((None, 0), (150, 20)):
        want, *sizes = kv_plain.attention(q[:keep], c, 0, [s for s in seqs if s[0]], d ** -0.5, window, first)
        for do in (BF, F32):
            out = torch.full((T, H, d), 7.0, dtype=do, device="cuda")
            call(q, tb, c, 0, d ** -0.5, window=window, first=first, out=out)
            assert bool((out[keep:] == 7).all())
            off = kv_plain.off_by(BF, do, max(n + s for n, s, _, _ in seqs), d, want, *sizes, decoded=True)      # the tiles take what the layout gives them
            err = (out[:keep].double().cpu() - want).abs()
            assert bool((err <= off).all()), (float((err / off).max()), float(err.max()))


def test_more_sequences_than_there_are_bits(monkeypatch):
    """Steps of thousands of sequences, some of them for the tiles: alone between others of few rows, and in a long run."""
    from krasis_b200 import seqops as ops
    monkeypatch.setattr(ops, "KV_TILES_FROM", 17)
    lens = [(5 if i in (7, 2050, 4099) or 3000 <= i < 3040 else 1, i * 7 % 40) for i in range(4100)]
    tb, seqs, pages = _step(lens, 16, 56)
    c = _cache(1, 64, 64, pages, "e4m3", 16, seed=57)
    q = torch.randn(tb.T, 4, 64, generator=_gen(58)).to(BF).cuda()
    want, *sizes = kv_plain.attention(q, c, 0, seqs, 0.125)
    got = ops.kv_attn(q, tb, c, 0, 0.125)
    off = kv_plain.off_by(BF, BF, 45, 64, want, *sizes, decoded=True)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= off).all()), (float((err / off).max()), float(err.max()))


@pytest.mark.parametrize("dq", [BF, F32])
@pytest.mark.parametrize("H,G,d,dv", [(16, 2, 128, 128), (6, 2, 256, 256), (8, 2, 48, 32)])
def test_queries_at_odd_offsets(dq, H, G, d, dv, forms):  # noqa: F811
    """Queries as part of a projection, at addresses that hold no four of them whole, heads apart by more than their numbers."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 300), (40, 200)], 64, 80)
    c = _cache(G, d, dv, pages, "e4m3", seed=81)
    proj = torch.randn(tb.T, 3 + H * (d + 5), generator=_gen(82)).to(dq).cuda()
    q = proj[:, 3:].unflatten(1, (H, d + 5))[..., :d]
    known = None
    for do in (BF, F32):
        for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, d ** -0.5, dtype=do)):
            known = _check(got, q, c, seqs, known=known, scale=d ** -0.5)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("H,G,d,dv", [(16, 2, 128, 128), (8, 2, 256, 256), (24, 8, 192, 128)])
def test_each_sequence_by_the_bound_of_its_kernel(fmt, H, G, d, dv, monkeypatch):
    """Codes and scales are held whole where a sequence has few rows, beside others on tiles or alone: the rounding of decoded numbers belongs to the tiles' sequences."""
    from krasis_b200 import seqops as ops
    lens = [(1, 700), (50, 300), (2, 33), (1, 2500), (30, 900)]
    tb, seqs, pages = _step(lens, 64, 83)
    c = _cache(G, d, dv, pages, fmt, seed=84)
    q = torch.randn(tb.T, H, d, generator=_gen(85)).to(BF).cuda()
    for window, first in ((None, 0), (500, 4)):
        want, *sizes = kv_plain.attention(q, c, 0, seqs, d ** -0.5, window, first)
        for tiles_from in (17, 1 << 30):
            monkeypatch.setattr(ops, "KV_TILES_FROM", tiles_from)
            tb._kv, at = None, 0
            got = ops.kv_attn(q, tb, c, 0, d ** -0.5, window=window, first=first).double().cpu()
            for n, start in lens:
                rows = slice(at, at + n)
                off = kv_plain.off_by(BF, BF, n + start, d, want[rows], *(x[rows] for x in sizes), decoded=n * H // G >= tiles_from)
                err = (got[rows] - want[rows]).abs()
                assert bool((err <= off).all()), (n, start, tiles_from, float((err / off).max()))
                at += n
