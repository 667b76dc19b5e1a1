"""The 8-bit cache of ragged-batch serving: writing, reading, windowed attention with visible first tokens, trees of drafted tokens, moving an accepted path."""
import numpy as np
import pytest
import torch

from tests import kv_plain

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def waits():
    yield
    from krasis_b200 import seqops as ops
    ops.check_waits()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache(G, d, dv, pages, fmt, page_size=64, layers=1, seed=0, full=True):
    from krasis_b200.attention import CompactKVCache
    c = CompactKVCache(layers, G, d, dv, "cuda", max_pages=pages, fmt=fmt, page_size=page_size)
    if full:
        kv_plain.fill(c, _gen(seed))
    return c


def _step(lens, page_size, seed=0, spare=2, parents=None):
    """lens [(tokens, start)] -> (tables, seqs for kv_plain.attention, pages in the pool); pages in random order."""
    from krasis_b200 import seqops as ops
    need = [(n + start + page_size - 1) // page_size for n, start in lens]
    order, at, entries, seqs = torch.randperm(sum(need) + spare, generator=_gen(seed)).tolist(), 0, [], []
    for i, ((n, start), k) in enumerate(zip(lens, need)):
        pages = order[at:at + k]
        at += k
        entries.append(([0] * n, start, i, pages) + ((parents[i],) if parents else ()))
        seqs.append((n, start, pages, parents[i] if parents else None))
    return (ops.DraftTables if parents else ops.StepTables)(entries, "cuda"), seqs, sum(need) + spare


@pytest.fixture
def forms(monkeypatch):
    """Runs a call by the library's choice of kernels and with every sequence of more than 16 rows per kv head on the tiles of the tensor cores (bf16 results)."""
    from krasis_b200 import seqops as ops

    def both(tb, call):
        for rows in (0, 17):
            monkeypatch.setattr(ops, "KV_TILES_FROM", rows)
            tb._kv = None
            yield call()
    return both


def _check(got, q, cache, seqs, layer=0, known=None, **kw):
    want, *sizes = known = known or kv_plain.attention(q, cache, layer, seqs, **kw)
    keys = max(n + s for n, s, _, _ in seqs)
    off = kv_plain.off_by(q.dtype, got.dtype, keys, cache.dim, want, *sizes, decoded=max(n for n, _, _, _ in seqs) * q.shape[1] // cache.num_kv_heads > 16)
    err = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= off).all()), (float((err / off).max()), float(err.max()))
    return known


# ------------------------------------------------------------------------------------------------ writing and reading

def _written(cache, seqs, k, v, before):
    """The whole pools as they should be after a write of k, v [T, G, n]."""
    want = [t.cpu().float().double().numpy().copy() if i < 2 else t.cpu().numpy().copy() for i, t in enumerate(before)]
    for x, (c, s) in ((k, (0, 2)), (v, (1, 3))):
        codes, scales = kv_plain.quantised(x.float().cpu().numpy(), cache.fmt)
        at = 0
        for n, start, pages, _ in seqs:
            for i in range(n):
                p, o = pages[(start + i) // cache.page_size], (start + i) % cache.page_size
                want[c][0, p, :, o], want[s][0, p, :, o] = codes[at], scales[at]
                at += 1
    return want


def _pools(cache):
    return [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


def _same_pools(cache, want):
    for t, w in zip(_pools(cache), want):
        got = t.cpu().float().double().numpy() if t.dim() == 5 else t.cpu().numpy()
        np.testing.assert_array_equal(got, w)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("G,d,dv,page_size,lens", [
    (2, 128, 128, 64, [(1, 0), (1, 63), (1, 64), (5, 126)]), (3, 64, 256, 16, [(37, 5)]), (1, 16, 48, 32, [(3, 31), (70, 0)]), (8, 192, 128, 128, [(1, 1000)]),
    (4, 256, 80, 1024, [(2, 1023)]),
])
def test_write(fmt, dtype, G, d, dv, page_size, lens):
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step(lens, page_size, 1)
    c, g = _cache(G, d, dv, pages, fmt, page_size), _gen(2)
    proj = (torch.randn(tb.T, 7 + G * (d + dv), generator=g) * torch.exp(2 * torch.randn(tb.T, 1, generator=g))).to(dtype).cuda()      # rows at odd offsets
    k, v = proj[:, 7:7 + G * d].view(tb.T, G, d), proj[:, 7 + G * d:].view(tb.T, G, dv)
    want = _written(c, seqs, k, v, _pools(c))
    ops.kv_write(k, v, tb, c, 0)
    _same_pools(c, want)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_hard_rows(fmt):
    """Rows of zeros, of smallest and largest numbers, with numbers that are not finite, and quotients on or next to the middle of two codes."""
    from krasis_b200 import seqops as ops
    d, rows = 64, []
    base = torch.randn(d, generator=_gen(3))
    for size in (0.0, 1e-45, 3e-44, 1e-40, 1.1754944e-38, 1e-30, 1e-20, 0.9e-20, 1.0, 1e20, 1e38):
        rows.append(base * size)
    rows += [torch.full((d,), torch.finfo(F32).max), torch.full((d,), -1e-45), -torch.zeros(d)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = base.clone()
        r[17] = bad
        rows.append(r)
    for top in (127.0, 448.0, 449.0, 1.75, 1.7500001, 7.0, 3.14159):
        halves = torch.arange(d) * (top / 127) + top / 254 if fmt == "int8" else torch.exp2(torch.arange(d) / 8.0 - 6) * 1.0625
        for jog in (0, 1, -1):
            r = halves.clone().clamp(max=top).numpy()
            if jog:
                r = np.nextafter(r, np.float32(jog * 1e38), dtype=np.float32)
            r = torch.from_numpy(r).clone()
            r[0] = top
            r[1::2] *= -1
            rows.append(r)
    x = torch.stack(rows)[:, None].cuda()
    tb, seqs, pages = _step([(len(rows), 9)], 64)
    c = _cache(1, d, d, pages, fmt)
    want = _written(c, seqs, x, -x, _pools(c))
    ops.kv_write(x, -x, tb, c, 0)
    _same_pools(c, want)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("G,d,dv,page_size,first,count", [(2, 128, 128, 64, 0, 200), (1, 16, 256, 16, 33, 1), (5, 96, 48, 32, 100, 0), (4, 256, 64, 128, 127, 129)])
def test_read(fmt, dtype, G, d, dv, page_size, first, count):
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 5), (1, first + count)], page_size, 4)
    c = _cache(G, d, dv, pages, fmt, page_size, layers=2)
    k, v = ops.kv_read(tb, 1, first, count, c, 1, dtype=dtype)
    assert k.shape == (count, G, d) and v.shape == (count, G, dv) and k.dtype == dtype
    for got, x in zip((k, v), kv_plain.held(c, 1)):
        want = x[seqs[1][2]].transpose(1, 2).reshape(-1, G, x.shape[-1])[first:first + count]
        # the product of an 8-bit code and a 24-bit scale is rounded to fp32 and that to bfloat16
        off = want.abs() * (2.0 ** -24 + (2.0 ** -8 if dtype == BF else 0.0))
        assert bool(((got.double().cpu() - want).abs() <= off).all())


# ------------------------------------------------------------------------------------------------ attention

SIZES = [(16, 2, 128, 128), (4, 4, 64, 64), (14, 2, 96, 96), (24, 8, 192, 128), (8, 1, 128, 256), (6, 2, 256, 256), (2, 1, 16, 240), (32, 1, 208, 16)]
STEPS = {"one": [(1, 0)], "few": [(1, 63), (1, 64), (1, 300)], "ragged": [(1, 0), (1, 700), (1, 15), (1, 16), (1, 2000)],
         "portions": [(37, 0), (1, 100), (90, 333)], "long": [(130, 1200)], "many keys": [(1, 9000)]}


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("H,G,d,dv", SIZES)
@pytest.mark.parametrize("step", sorted(STEPS))
def test_attention(fmt, H, G, d, dv, step, forms):
    from krasis_b200 import seqops as ops
    i = SIZES.index((H, G, d, dv)) + sorted(STEPS).index(step)
    page_size = (64, 16, 128)[i % 3]
    tb, seqs, pages = _step(STEPS[step], page_size, i)
    c = _cache(G, d, dv, pages, fmt, page_size, layers=2, seed=i)
    for window, first in ((None, 0), (100, 4), (17, 300)):
        for dq in (F32, BF):
            q, known = torch.randn(tb.T, H, d, generator=_gen(i)).to(dq).cuda(), None
            for do in (F32, BF):
                for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 1, d ** -0.5, window=window, first=first, dtype=do)):
                    known = _check(got, q, c, seqs, 1, known=known, scale=d ** -0.5, window=window, first=first)


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (1, 64), (16, 16), (15, 17), (5000, 3), (2, 100000)])
def test_windows(window, first, forms):
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 0), (50, 0), (1, 31), (1, 500), (20, 90)], 16, 5)
    c = _cache(2, 64, 64, pages, "int8", 16)
    q = torch.randn(tb.T, 6, 64, generator=_gen(6)).cuda()
    known = None
    for do in (BF, F32):
        for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, 0.125, window=window, first=first, dtype=do)):
            known = _check(got, q, c, seqs, known=known, scale=0.125, window=window, first=first)


def test_sinks_and_scales(forms):
    """Scores far apart, a negative scale, sinks below and above all scores, rows of values whose scales are 1e8 apart."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(3, 400), (1, 3000)], 64, 7)
    c = _cache(2, 128, 128, pages, "e4m3")
    c.v_scale[0, :, 0] *= torch.exp2(torch.randint(-13, 13, c.v_scale[0, :, 0].shape, generator=_gen(8)).float()).cuda()
    sinks = torch.linspace(-30, 30, 8).cuda()
    q = (torch.randn(tb.T, 8, 128, generator=_gen(9)) * torch.exp2(torch.randint(-6, 3, (tb.T, 8, 1), generator=_gen(10)).float())).cuda()
    for scale in (0.09, -0.09, 1.0, 0.0):
        for s in (None, sinks):
            got = ops.kv_attn(q, tb, c, 0, scale, sinks=s, dtype=F32)
            _check(got, q, c, seqs, scale=scale, sinks=s)
    # on tiles a value row keeps its bits down to 2^-21 of its tile's largest scale
    tb, seqs, pages = _step([(13, 400), (40, 21), (1, 3000)], 64, 7)
    c = _cache(2, 128, 128, pages, "int8")
    c.v_scale[0, :, 0] *= torch.exp2(torch.randint(-6, 6, c.v_scale[0, :, 0].shape, generator=_gen(8)).float()).cuda()
    q = (torch.randn(tb.T, 8, 128, generator=_gen(9)) * torch.exp2(torch.randint(-6, 3, (tb.T, 8, 1), generator=_gen(10)).float())).cuda()
    for scale in (0.09, -0.09, 0.0):
        for s in (None, sinks):
            known = None
            for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, scale, sinks=s, dtype=BF)):
                known = _check(got, q, c, seqs, known=known, scale=scale, sinks=s)


@pytest.mark.parametrize("H,G,d,dv", [(16, 2, 128, 128), (8, 2, 256, 256), (14, 2, 96, 96)])
def test_one_key_far_above_the_others(H, G, d, dv, forms):
    """Keys whose scores lie 100 powers of e above all others come late, twice: what was summed before counts for nothing then."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(20, 1000), (1, 700)], 64, 29)
    c = _cache(G, d, dv, pages, "int8")
    q = torch.randn(tb.T, H, d, generator=_gen(30)).cuda()
    for s, (n, start, pl, _) in enumerate(seqs):
        t = 0 if s == 0 else 20
        for g in range(G):
            for j, gain in ((300, 60.0), (start - 70, 100.0)):
                x = q[t, g * (H // G)] * gain / float(q[t, g * (H // G)].square().sum()) / d ** -0.5
                top = float(x.abs().max())
                c.k[0, pl[j // 64], g, j % 64] = torch.round(x * 127 / top).to(torch.int8)
                c.k_scale[0, pl[j // 64], g, j % 64] = top / 127
    known = None
    for do in (F32, BF):
        for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, d ** -0.5, dtype=do)):
            known = _check(got, q, c, seqs, known=known, scale=d ** -0.5)


@pytest.mark.parametrize("lens,H,G,d", [([(1, 30000), (1, 0), (1, 17), (1, 4000), (1, 900)], 16, 8, 64), ([(1, 20000 + 97 * i) for i in range(3)], 12, 12, 128),
                                        ([(2, 7000)] * 5, 16, 4, 256), ([(1, 50000)], 64, 4, 128), ([(1, 9000 * (i % 3)) for i in range(40)], 7, 7, 128)])
def test_many_keys(lens, H, G, d):
    """Requests with so many keys that these are cut evenly over the GPU, wherever the ends lie in the requests."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step(lens, 64, 3)
    c = _cache(G, d, d, pages, "int8")
    q = torch.randn(tb.T, H, d, generator=_gen(1)).cuda()
    for window, first in ((None, 0), (8000, 5)):
        known = None
        for do in (F32, BF):
            known = _check(ops.kv_attn(q, tb, c, 0, d ** -0.5, dtype=do, window=window, first=first), q, c, seqs, known=known, scale=d ** -0.5, window=window, first=first)


def test_a_row_is_the_same_however_it_is_cut(monkeypatch):
    """One request alone, beside many others, as a single token and within a portion: the same numbers up to roundings."""
    from krasis_b200 import seqops as ops
    lens = [(1, 3000)] + [(1, 100 * i) for i in range(30)] + [(70, 900)]
    tb, seqs, pages = _step(lens, 64, 31)
    c = _cache(2, 128, 128, pages, "e4m3")
    q = torch.randn(tb.T, 16, 128, generator=_gen(32)).cuda()
    whole = ops.kv_attn(q, tb, c, 0, 0.09, dtype=F32)
    for i in (0, 7, 31):
        n, start, pl, _ = seqs[i]
        at = sum(x for x, _ in lens[:i])
        alone = ops.kv_attn(q[at:at + n], ops.StepTables([([0] * n, start, 0, pl)], "cuda"), c, 0, 0.09, dtype=F32)
        assert float((alone - whole[at:at + n]).abs().max()) < 1e-5 * float(whole.abs().max())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("lens,H,G,d", [([(1, 130), (40, 21), (1, 700)], 8, 2, 64), ([(150, 77)], 16, 2, 128)])
def test_rows_that_are_not_numbers(fmt, lens, H, G, d, forms):
    """A token with a NaN in its key (or an infinity in its value) makes NaN for the tokens and heads that see it and for no others."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step(lens, 16, 11)
    g = _gen(12)
    for which in (0, 1):
        c = _cache(G, d, d, pages, fmt, 16, seed=3)
        k, v = (torch.randn(tb.T, G, d, generator=g).cuda() for _ in range(2))
        s = max(range(len(lens)), key=lambda i: lens[i][0])            # in the middle of the longest portion
        at = sum(n for n, _ in lens[:s]) + lens[s][0] // 2
        (k, v)[which][at, 1, 3] = float("nan") if which == 0 else float("inf")
        ops.kv_write(k, v, tb, c, 0)
        q = torch.randn(tb.T, H, d, generator=g).cuda()
        for window, first in ((None, 0), (9, 2)):
            for do in (BF, F32):
                see = torch.zeros(tb.T, H, dtype=torch.bool)
                last = sum(n for n, _ in lens[:s + 1]) if window is None else min(at + window, sum(n for n, _ in lens[:s + 1]))
                see[at:last, H // G:2 * (H // G)] = True
                for got in forms(tb, lambda: ops.kv_attn(q, tb, c, 0, 0.1, window=window, first=first, dtype=do).cpu()):
                    assert torch.equal(torch.isnan(got).all(-1), see) and bool(torch.isfinite(got[~see]).all())


def test_what_nobody_sees_changes_nothing(forms):
    """Rows behind the sequences, ahead of the windows and in strange pages hold codes of another life and NaN scales: the bits stay."""
    from krasis_b200 import seqops as ops
    lens = [(1, 777), (30, 200), (1, 3), (200, 50)]
    tb, seqs, pages = _step(lens, 64, 13)
    for fmt in ("e4m3", "int8"):
        c = _cache(2, 128, 128, pages, fmt, seed=1)
        q = torch.randn(tb.T, 16, 128, generator=_gen(14)).cuda()
        calls = [lambda do=do: list(forms(tb, lambda: ops.kv_attn(q, tb, c, 0, 0.09, window=60, first=5, dtype=do))) for do in (BF, F32)]
        before = [f() for f in calls]
        mark = torch.ones(pages, 64, dtype=torch.bool)
        for n, start, pl, _ in seqs:
            for j in list(range(5)) + list(range(max(0, start - 59), start + n)):
                if j < start + n:
                    mark[pl[j // 64], j % 64] = False
        mark = mark.cuda()
        for sc in (c.k_scale, c.v_scale):
            sc[0].transpose(1, 2)[mark] = float("nan")
        for a, f in zip(before, calls):
            assert all(torch.equal(x, y) for x, y in zip(a, f()))


def test_pages_outside_the_pool():
    """A page number that the pool does not have holds nothing: no write goes there, and its rows are not seen."""
    from krasis_b200 import seqops as ops
    for bad in (6, 1 << 20, -1, -(1 << 31)):
        tb = ops.StepTables([([0] * 3, 190, 0, [5, 3, 1, 0]), ([0], 10, 1, [2])], "cuda")
        tb.pages[1] = bad                                  # positions 64 .. 127 of the first sequence
        c = _cache(2, 64, 64, 6, "int8", seed=2)
        q = torch.randn(tb.T, 4, 64, generator=_gen(15)).cuda()
        got = ops.kv_attn(q, tb, c, 0, 0.125, dtype=F32)
        k, v = kv_plain.held(c, 0)
        for t in range(3):
            rows = [j for j in range(190 + t + 1) if not 64 <= j < 128]
            at = torch.tensor([[5, 3, 1, 0][j // 64] for j in rows]), torch.tensor([j % 64 for j in rows])
            for h in range(4):
                kk, vv = k[at[0], h // 2, at[1]], v[at[0], h // 2, at[1]]
                w = torch.softmax(kk @ q[t, h].double().cpu() * 0.125, 0)
                assert float((got[t, h].double().cpu() - w @ vv).abs().max()) < 1e-4
        x = torch.ones(tb.T, 2, 64, device="cuda")
        tb.pages[2] = bad                                  # now the new rows, 190 and 191, have no page either
        before = _pools(c)
        ops.kv_write(x, x, tb, c, 0)
        before[0][0, 0, :, 0], before[1][0, 0, :, 0] = 127, 127         # row 192
        before[2][0, 0, :, 0], before[3][0, 0, :, 0] = 1 / 127, 1 / 127
        before[0][0, 2, :, 10], before[1][0, 2, :, 10] = 127, 127
        before[2][0, 2, :, 10], before[3][0, 2, :, 10] = 1 / 127, 1 / 127
        for a, b in zip(before, _pools(c)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("d,dv", [(64, 64), (192, 128), (256, 256)])
@pytest.mark.parametrize("tokens", [40, 8])
def test_pages_outside_the_pool_on_tiles(d, dv, tokens, monkeypatch):
    """The same where the tensor cores' tiles take the rows: a missing page's rows have no weight, not even that of a score of 0."""
    from krasis_b200 import seqops as ops
    monkeypatch.setattr(ops, "KV_TILES_FROM", 1)
    for bad in (6, -1):
        pages = [5, 3, 1, 0]
        tb = ops.StepTables([([0] * tokens, 190, 0, pages)], "cuda")
        tb.pages[1] = bad                                  # positions 64 .. 127
        c = _cache(2, d, dv, 6, "int8", seed=2)
        q = (torch.randn(tokens, 8, d, generator=_gen(15)) - 0.5).to(BF).cuda()
        (k, v), codes = kv_plain.held(c, 0), c.v[0].double().abs().cpu()
        for window, first in ((None, 0), (150, 70)):
            got = ops.kv_attn(q, tb, c, 0, 0.125, window=window, first=first)
            for t in range(tokens):
                rows = [j for j in range(190 + t + 1) if not 64 <= j < 128 and (window is None or 190 + t - j < window or j < first)]
                at = torch.tensor([pages[j // 64] for j in rows]), torch.tensor([j % 64 for j in rows])
                for h in range(8):
                    kk, vv, x = k[at[0], h // 4, at[1]], v[at[0], h // 4, at[1]], q[t, h].double().cpu()
                    w = torch.softmax(kk @ x * 0.125, 0)
                    off = kv_plain.off_by(BF, BF, 256, d, w @ vv, w @ vv.abs(), (kk.abs() @ x.abs()).max() * 0.125,
                                          (w * c.v_scale[0].double().cpu()[at[0], h // 4, at[1]]).max() * codes[at[0], h // 4, at[1]].sum(0), decoded=True)
                    assert bool(((got[t, h].double().cpu() - w @ vv).abs() <= off).all())


def test_rows_behind_the_last_sequence():
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(2, 40), (3, 7)], 64, 16)
    tb.cu[2] = 4                                           # the last row belongs to nobody
    c = _cache(2, 64, 64, pages, "e4m3")
    before, x = _pools(c), torch.randn(5, 2, 64, generator=_gen(17)).cuda()
    seqs[1] = (2,) + seqs[1][1:]
    want = _written(c, seqs, x[:4], x[:4], before)
    ops.kv_write(x, x, tb, c, 0)
    _same_pools(c, want)
    q, out = torch.randn(5, 4, 64, generator=_gen(18)).cuda(), torch.full((5, 4, 64), 7.0, device="cuda")
    ops.kv_attn(q, tb, c, 0, 0.125, out=out)
    assert bool((out[4] == 7).all())
    _check(out[:4], q[:4], c, seqs, scale=0.125)


def test_rows_past_two_to_the_31():
    """Pools of more than 2^31 numbers, pages at their end."""
    from krasis_b200 import seqops as ops
    from krasis_b200.attention import CompactKVCache
    pages = 8400
    c = CompactKVCache(1, 1, 256, 256, "cuda", max_pages=pages, fmt="int8", page_size=1024)
    tb = ops.StepTables([([0] * 4, 1022, 0, [pages - 1, pages - 2])], "cuda")
    g = _gen(19)
    k, v = (torch.randn(4, 1, 256, generator=g).cuda() for _ in range(2))
    ops.kv_write(k, v, tb, c, 0)
    q = torch.randn(4, 2, 256, generator=g).cuda()
    got = ops.kv_attn(q, tb, c, 0, 0.06, window=4, dtype=F32)
    kk, vv = ops.kv_read(tb, 0, 1022, 4, c, 0, dtype=F32)
    for t in range(4):
        lo = 1022 + t - 3
        keep = [j for j in range(4) if lo <= 1022 + j <= 1022 + t]
        zeros = 4 - len(keep)                              # rows ahead of the portion hold zeros: score 0, value 0
        for h in range(2):
            x = torch.cat([kk[keep, 0].double() @ q[t, h].double() * 0.06, torch.zeros(zeros, device="cuda", dtype=torch.float64)])
            w = torch.softmax(x, 0)[:len(keep)]
            assert float((got[t, h].double() - w @ vv[keep, 0].double()).abs().max()) < 1e-5
    for x, y in ((k, kk), (v, vv)):
        assert float((x - y).abs().max()) <= float(x.abs().max()) / 254 * 1.01


# ------------------------------------------------------------------------------------------------ trees

def _tree(n, seed, span):
    g = np.random.RandomState(seed)
    return [max(-1, i - 1 - int(g.randint(0, span))) for i in range(n)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("H,G,d,dv", [(16, 2, 128, 128), (4, 4, 64, 64), (24, 8, 192, 128), (32, 1, 128, 256), (6, 2, 256, 256)])
@pytest.mark.parametrize("lens", [[(1, 0)], [(16, 700)], [(5, 0), (33, 64), (1, 500), (64, 90)], [(70, 1000), (300, 40)]])
def test_tree(fmt, H, G, d, dv, lens, forms):
    from krasis_b200 import seqops as ops
    i = H + len(lens)
    tb, seqs, pages = _step(lens, (64, 16)[i % 2], i, parents=[_tree(n, i + n, 4) for n, _ in lens])
    c = _cache(G, d, dv, pages, fmt, (64, 16)[i % 2], layers=2, seed=i)
    for window, first in ((None, 0), (30, 7), (2, 0)):
        for dq, do in ((F32, BF), (BF, BF), (F32, F32)):
            q = torch.randn(tb.T, H, d, generator=_gen(i)).to(dq).cuda()
            known = None
            for got in forms(tb, lambda: ops.kv_tree_attn(q, tb, c, 1, d ** -0.5, window=window, first=first, dtype=do)):
                known = _check(got, q, c, seqs, 1, known=known, scale=d ** -0.5, window=window, first=first)


def test_tree_tables():
    from krasis_b200 import seqops as ops
    tb = ops.DraftTables([([1, 2, 3, 4], 10, 0, [0], [-1, 0, 0, 2]), ([5] * 40, 3, 1, [1], [-1] + list(range(39)))], "cuda")
    assert tb.positions[:4].tolist() == [10, 11, 11, 12] and tb.rows[:4].tolist() == [10, 11, 12, 13] and tb.words == 2
    assert tb.bits[:4, 0].tolist() == [1, 3, 5, 13] and tb.bits[:4, 1].tolist() == [0] * 4
    assert tb.positions[4:].tolist() == list(range(3, 43))
    assert [b & 0xFFFFFFFF for b in tb.bits[43].tolist()] == [0xFFFFFFFF, 0xFF]


def test_chain_is_a_portion():
    """A tree without branches sees what a portion sees."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(40, 333), (7, 0)], 64, 20)
    dt = ops.DraftTables([([0] * n, s, 0, p, list(range(-1, n - 1))) for n, s, p, _ in seqs], "cuda")
    c = _cache(2, 128, 128, pages, "int8")
    q = torch.randn(tb.T, 8, 128, generator=_gen(21)).cuda()
    for window in (None, 50):
        a, b = ops.kv_attn(q, tb, c, 0, 0.1, window=window, first=3, dtype=F32), ops.kv_tree_attn(q, dt, c, 0, 0.1, window=window, first=3, dtype=F32)
        assert float((a - b).abs().max()) < 1e-4 * float(a.abs().max())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_keep(fmt):
    from krasis_b200 import seqops as ops
    lens = [(9, 60), (20, 10), (1, 500), (12, 0), (6, 63)]
    tb, seqs, pages = _step(lens, 16, 22, parents=[_tree(n, n, 3) for n, _ in lens])
    paths = [[0, 2, 3, 8, -1], [1, 5, 6, 7, 19], [0, -1, -1, -1, -1], [-1, 3, 4, 5, 6], [0, 4, 3, 5, 5]]
    want_paths = [[0, 2, 3, 8], [1, 5, 6, 7, 19], [0], [], [0, 4]]
    c = _cache(3, 96, 48, pages, fmt, 16, layers=3)
    want = _pools(c)
    for (n, start, pl, _), path in zip(seqs, want_paths):
        frm = [(pl[(start + p) // 16], (start + p) % 16) for p in path]
        for t in want:
            rows = [t[:, p, :, o].clone() for p, o in frm]
            for i, r in enumerate(rows):
                t[:, pl[(start + i) // 16], :, (start + i) % 16] = r
    ops.kv_keep(tb, torch.tensor(paths, dtype=torch.int32, device="cuda"), c)
    for a, b in zip(want, _pools(c)):
        assert torch.equal(a.view(torch.uint8) if a.dtype != F32 else a, b.view(torch.uint8) if b.dtype != F32 else b)
    ops.kv_keep(tb, torch.zeros(5, 0, dtype=torch.int32, device="cuda"), c)
    for bad in ([[9, -1]] * 5, [[99, 3]] * 5, [[-7, 1]] * 5):          # of the sequences of 20 and 12 tokens the first moves row 9
        want = _pools(c)
        for (n, start, pl, _) in seqs:
            if bad[0][0] == 9 and n > 9:
                for t in want:
                    t[:, pl[start // 16], :, start % 16] = t[:, pl[(start + 9) // 16], :, (start + 9) % 16].clone()
        ops.kv_keep(tb, torch.tensor(bad, dtype=torch.int32, device="cuda"), c)
        for a, b in zip(want, _pools(c)):
            assert torch.equal(a.view(torch.uint8) if a.dtype != F32 else a, b.view(torch.uint8) if b.dtype != F32 else b)


# ------------------------------------------------------------------------------------------------ together

@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_request_with_drafts(fmt):
    """Two requests: prompts in portions, then trees of drafted tokens of which a path is kept, then single tokens; every result against a plain cache that holds what was
    written.  Pages come from the cache's free list."""
    from krasis_b200 import seqops as ops
    from krasis_b200.attention import CompactKVCache, SequenceKVState
    H, G, d, ps = 8, 2, 128, 16
    c = CompactKVCache(2, G, d, d, "cuda", max_pages=40, fmt=fmt, page_size=ps)
    states, g = [SequenceKVState(c, i) for i in range(2)], _gen(23)

    def run(lens, parents=None):
        entries = []
        for st, n in zip(states, lens):
            st.ensure_capacity(n)
            entries.append(([0] * n, st.seq_len, 0, st.pages))
        tb = ops.DraftTables([e + (p,) for e, p in zip(entries, parents)], "cuda") if parents else ops.StepTables(entries, "cuda")
        seqs = [(n, st.seq_len, list(st.pages), parents[i] if parents else None) for i, (st, n) in enumerate(zip(states, lens))]
        for layer in range(2):
            k, v = (torch.randn(tb.T, G, d, generator=g).cuda() for _ in range(2))
            ops.kv_write(k, v, tb, c, layer)
            q = torch.randn(tb.T, H, d, generator=g).cuda()
            for window, first in ((None, 0), (24, 3)):
                call = ops.kv_tree_attn if parents else ops.kv_attn
                _check(call(q, tb, c, layer, 0.09, window=window, first=first, dtype=BF), q, c, seqs, layer, scale=0.09, window=window, first=first)
        return tb

    run([40, 7])
    for st, n in zip(states, (40, 7)):
        st.advance(n)
    run([21, 1])
    for st, n in zip(states, (21, 1)):
        st.advance(n)
    for r in range(3):
        lens = [9 + r, 14]
        parents = [_tree(n, n + r, 3) for n in lens]
        tb = run(lens, parents)
        paths = []
        for ps_ in parents:                                # the longest path of each tree
            depth, best = [], 0
            for i, p in enumerate(ps_):
                depth.append(depth[p] + 1 if p >= 0 else 0)
                best = i if depth[i] > depth[best] else best
            path = [best]
            while ps_[path[0]] >= 0:
                path.insert(0, ps_[path[0]])
            paths.append(path)
        kept = [[x.clone() for x in ops.kv_read(tb, s, st.seq_len, n, c, 1)] for s, (st, n) in enumerate(zip(states, lens))]
        P = max(map(len, paths))
        ops.kv_keep(tb, torch.tensor([p + [-1] * (P - len(p)) for p in paths], dtype=torch.int32, device="cuda"), c)
        for s, (st, path) in enumerate(zip(states, paths)):
            for x, y in zip(ops.kv_read(tb, s, st.seq_len, len(path), c, 1), kept[s]):
                assert torch.equal(x, y[path])
            st.advance(len(path))
        run([1, 1])
        for st in states:
            st.advance(1)
    ops.check_waits()


def test_captured_decode():
    """A captured step runs again with later positions and other pages, beside a second captured step and eager calls on another stream."""
    from krasis_b200 import seqops as ops
    from krasis_b200.graphs import capture
    H, G, d, S = 8, 2, 128, 3
    c, g = _cache(G, d, d, 64, "int8", 16), _gen(24)
    pages = torch.randperm(64, generator=g).tolist()
    lists = [pages[0:16], pages[16:32], pages[32:48]]
    k, v, q = (torch.randn(S, h, d, generator=g).cuda() for h in (G, G, H))
    n = 3 * S + (S + 1) + S + S * 16

    def tables(starts, buf):
        return ops.StepTables([([0], s, i, lists[i]) for i, s in enumerate(starts)], "cuda", device_buf=buf)

    def step(tb, window):
        ops.kv_write(k, v, tb, c, 0)
        return ops.kv_attn(q, tb, c, 0, 0.09, window=window, first=2, dtype=F32)
    bufs = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2)]
    tbs = [tables([5, 0, 9], b) for b in bufs]
    graphs = [capture(lambda tb=tb, w=w: step(tb, w), "cuda") for tb, w in zip(tbs, (None, 40))]
    other = torch.cuda.Stream()
    for starts in ([5, 0, 9], [250, 17, 100], [31, 255, 255]):
        kept = [tables(starts, b) for b in bufs]
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        seqs = [(1, s, lists[i], None) for i, s in enumerate(starts)]
        for (gr, out), w in zip(graphs, (None, 40)):
            _check(out, q, c, seqs, scale=0.09, window=w, first=2)
        del kept
        with torch.cuda.stream(other):
            eager = ops.kv_attn(q, ops.StepTables([([0], s, i, lists[i]) for i, s in enumerate(starts)], "cuda"), c, 0, 0.09, window=40, first=2, dtype=F32)
        other.synchronize()
        _check(eager, q, c, seqs, scale=0.09, window=40, first=2)


@pytest.mark.parametrize("tree", [False, True])
def test_captured_portions(tree, monkeypatch):
    """A captured step of portions or trees (tiles of the tensor cores, pieces and their join) runs again with later positions."""
    from krasis_b200 import seqops as ops
    from krasis_b200.graphs import capture
    monkeypatch.setattr(ops, "KV_TILES_FROM", 17)
    H, G, d, ns = 8, 2, 128, (24, 9)
    c, g = _cache(G, d, d, 64, "int8", 16), _gen(33)
    pages = torch.randperm(64, generator=g).tolist()
    lists, T = [pages[0:32], pages[32:64]], sum(ns)
    q = torch.randn(T, H, d, generator=g).cuda()
    parents = [_tree(n, n, 3) for n in ns]
    buf = torch.zeros(3 * T + 3 + 2 + 2 * 32, dtype=torch.int32, device="cuda")
    draft = torch.zeros(2 * T, dtype=torch.int32, device="cuda")

    def tables(starts):
        e = [([0] * n, s, i, lists[i]) for i, (n, s) in enumerate(zip(ns, starts))]
        return ops.DraftTables([x + (p,) for x, p in zip(e, parents)], "cuda", device_buf=buf, draft_buf=draft) if tree else ops.StepTables(e, "cuda", device_buf=buf)
    call = ops.kv_tree_attn if tree else ops.kv_attn
    tb = tables((3, 40))
    graph, out = capture(lambda: call(q, tb, c, 0, 0.09, window=200, first=3, dtype=BF), "cuda")
    for starts in ((3, 40), (480, 0), (0, 500)):
        kept = tables(starts)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, c, [(n, s, lists[i], parents[i] if tree else None) for i, (n, s) in enumerate(zip(ns, starts))], scale=0.09, window=200, first=3)
        del kept


def test_captured_many_keys():
    """A captured decode step whose page lists have room for many keys: cut evenly by whatever the positions are when it runs."""
    from krasis_b200 import seqops as ops
    from krasis_b200.graphs import capture
    H, G, d, S, room = 16, 8, 64, 2, 400
    c, g = _cache(G, d, d, 2 * room, "e4m3", 64), _gen(34)
    lists = [list(range(0, room)), list(range(2 * room - 1, room - 1, -1))]
    q = torch.randn(S, H, d, generator=g).cuda()
    buf = torch.zeros(3 * S + S + 1 + S + S * room, dtype=torch.int32, device="cuda")
    tables = lambda starts: ops.StepTables([([0], s, i, lists[i]) for i, s in enumerate(starts)], "cuda", device_buf=buf)  # noqa: E731
    tb = tables((25000, 25000))
    graph, out = capture(lambda: ops.kv_attn(q, tb, c, 0, 0.1, dtype=F32), "cuda")
    for starts in ((25000, 25000), (0, 25599), (0, 0), (130, 7000)):
        kept = tables(starts)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, c, [(1, s, lists[i], None) for i, s in enumerate(starts)], scale=0.1)
        del kept


def test_two_streams_at_once():
    """Calls on two streams, each with its own results and workspaces, and tables that both read."""
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 6000), (1, 90), (60, 2000)], 64, 35)
    c = _cache(2, 128, 128, pages, "int8")
    q = torch.randn(tb.T, 16, 128, generator=_gen(36)).cuda()
    want = [ops.kv_attn(q * f, tb, c, 0, 0.09, dtype=do) for f, do in ((1.0, BF), (0.5, F32))]
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for i, (s, f, do) in enumerate(zip(streams, (1.0, 0.5), (BF, F32))):
            with torch.cuda.stream(s):
                got[i].append(ops.kv_attn(q * f, tb, c, 0, 0.09, dtype=do))
    torch.cuda.synchronize()
    for w, xs in zip(want, got):
        assert all(torch.equal(w, x) for x in xs)


def test_same_call_same_bits():
    from krasis_b200 import seqops as ops
    tb, seqs, pages = _step([(1, 5000), (1, 90), (33, 700)], 64, 25)
    c = _cache(2, 128, 128, pages, "e4m3")
    q = torch.randn(tb.T, 16, 128, generator=_gen(26)).cuda()
    for do in (BF, F32):
        a = ops.kv_attn(q, tb, c, 0, 0.09, dtype=do)
        for _ in range(5):
            assert torch.equal(a, ops.kv_attn(q, tb, c, 0, 0.09, dtype=do))
