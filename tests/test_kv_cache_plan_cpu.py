"""How the attention over the 8-bit cache plans its work, without a GPU: the workspace that a call asks for."""
import ctypes as C

import numpy as np
import pytest
import torch

from krasis_b200 import seqops as ops


def _workspace(lens, H, G, d, dv, dt_out=1, window=0, first=0, replayed=0, tiles_from=0, max_pages=None, page_size=64):
    """Bytes for a step of [(tokens, start)]."""
    pages = [(n + start + page_size - 1) // page_size for n, start in lens]
    first_rows = np.cumsum([0] + [n for n, _ in lens])
    layout = np.array([[r, n, start, p] for r, (n, start), p in zip(first_rows, lens, pages)], dtype=np.int32)
    cache = ops.KvCacheArgs(4096, 4096, 4096, 4096, 1, sum(pages), page_size, G, d, dv, 1)
    step = ops.KvStepArgs(4096, 4096, 4096, 4096, None, None, layout.ctypes.data, 0, int(first_rows[-1]), len(lens), max_pages or max(pages), replayed, 0, tiles_from)
    return ops.load().kb2_seq_kv_attn_workspace(C.byref(cache), C.byref(step), H, window, first, dt_out)


MB = 1 << 20


@pytest.mark.parametrize("H,G,decode,portion", [(64, 4, [30000], (4096, 0)), (64, 4, [60000], (8192, 0)), (64, 4, [500 + 950 * i for i in range(32)], (4096, 5001)), (16, 2, [30000], (2048, 0)),
                                                (64, 4, [1000000], (8192, 0)), (64, 4, [30000, 100, 200], (3000, 100)), (32, 32, [60000] * 4, (4096, 0))])
@pytest.mark.parametrize("replayed", [0, 1])
def test_mixed_steps_ask_for_what_is_cut(H, G, decode, portion, replayed):
    """A portion beside decoding requests: the partial results are those of the rows that are cut.  A decoded token's keys are cut into at most 64 pieces, or one for each 768
    groups of 16, so its rows have at most so many results of d numbers, a maximum and a sum; the portion has what it has alone."""
    lens, pages = [(1, n) for n in decode] + [portion], (max(decode + [sum(portion)]) + 64) // 64
    size = lambda lens: _workspace(lens, H, G, 128, 128, replayed=replayed, max_pages=pages)  # noqa: E731
    rows = len(decode) * H * max(64, (max(decode) + 1) // (16 * 768) + 2)
    assert size(lens) <= rows * 130 * 4 + size(lens[-1:]) + 64
    assert size(lens) <= size(lens[:-1]) + size(lens[-1:]) + 80 * MB


@pytest.mark.parametrize("lens", [[(1, 30000)] + [(1, 16)] * 63, [(1, 1000000)] + [(1, 100)] * 511, [(1, 500 * i + 1) for i in range(64)]])
def test_decoding_steps_ask_for_what_is_cut(lens):
    """Requests of very different lengths: partial results in proportion to the pieces there are, not to the longest request's times all rows.  Cut evenly there is a piece
    for each of the 296 blocks (or each 768 groups) and one for each tile and head, 16 rows each; in pieces of tiles at most 64 of each request that is longer than a 64th of the longest."""
    got = _workspace(lens, 64, 4, 128, 128)
    groups = [(1 + n + 30) // 16 for _, n in lens]          # wherever the first of them begins in its 16
    even = (max(296, (sum(groups) + 40 * len(lens)) * 4 // 768 + 1) + len(lens) * 4) * 16 * 130 * 4 + len(lens) * 4 * 8
    tiles = sum(64 * max(1, min(64, (64 * g + max(groups) - 1) // max(groups))) for g in groups) * 130 * 4
    assert got <= max(even, tiles) + 64


@pytest.mark.parametrize("lens", [[(1, 60000)], [(600, 5000), (1, 60000)], [(4096, 5001)]])
def test_fp32_results_ask_for_what_is_cut(lens):
    """Portions with fp32 results beside a long request: at most 64 pieces for the request, and none for a portion whose keys one piece holds (768 groups of 16)."""
    cut = sum(n * 64 * min(64, max(1, (n + start + 15) // 16 // 8)) for n, start in lens if n == 1 or n + start > 768 * 16)
    assert _workspace(lens, 64, 4, 128, 128, dt_out=0) <= max(cut, 296 * 16 + 64 * 4) * 130 * 4 + 1024


# ------------------------------------------------------------------------------------------------ steps without tokens

def _empty(positions=None, **kw):
    layout = np.array([[0, 0, 5, 1]], dtype=np.int32)
    cache = ops.KvCacheArgs(4096, 4096, 4096, 4096, 2, 6, 16, 2, 64, 32, 1)
    step = dict(positions=positions, seq_of=positions, cu=4096, pages=4096, rows=None, bits=None, layout=layout.ctypes.data, words=0, T=0, S=1, max_pages=1, replayed=0, device=0, tiles_from=0)
    step.update(kw)
    return cache, ops.KvStepArgs(**step), layout


def test_a_step_without_tokens_does_nothing():
    """Empty tensors have no address."""
    lib = ops.load()
    cache, step, keep = _empty()
    p, q = C.byref(cache), C.byref(step)
    assert lib.kb2_seq_kv_write(p, 0, q, None, 128, 64, None, 64, 32, 0, None) == 0
    assert lib.kb2_seq_kv_attn_workspace(p, q, 4, 0, 0, 1) == 0
    assert lib.kb2_seq_kv_attn(p, 0, q, None, 0, 256, 64, 4, 1.0, 0, 0, None, None, 0, None, 0, None) == 0
    assert lib.kb2_seq_kv_keep(p, q, 4096, 1, None) == 0
    assert lib.kb2_seq_kv_read(p, 0, q, 0, 0, 0, None, None, 0, None) == 0
    # what has tokens or bad arguments is refused as before
    assert lib.kb2_seq_kv_write(p, 2, q, None, 128, 64, None, 64, 32, 0, None) == 4 and lib.kb2_seq_kv_write(p, 0, q, None, 128, 64, None, 64, 32, 2, None) == 2
    assert lib.kb2_seq_kv_attn(p, 0, q, None, 0, 256, 64, 3, 1.0, 0, 0, None, None, 0, None, 0, None) == 2
    for kw in (dict(cu=None), dict(pages=None), dict(layout=None), dict(T=1), dict(T=1, positions=4096, seq_of=None)):
        cache, step, keep = _empty(**kw)
        assert lib.kb2_seq_kv_write(C.byref(cache), 0, C.byref(step), 4096, 128, 64, 4096, 64, 32, 0, None) == 2


def test_rows_are_read_through_tables_without_tokens():
    """Tables that were made to read a sequence back: what they do not have is not asked for, what the pages do not hold is refused."""
    cache, step, keep = _empty()
    assert ops.load().kb2_seq_kv_read(C.byref(cache), 0, C.byref(step), 0, 0, 17, 4096, 4096, 0, None) == 4


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")
@pytest.mark.parametrize("lens,do,kw", [([(1, 199999)], 0, {}), ([(40, 3000), (1, 5000)], 1, {"tiles_from": 17}), ([(1, 9000)] * 40, 1, {})])
def test_a_workspace_that_is_too_small_is_refused(lens, do, kw):
    """Ahead of everything that needs a GPU."""
    lib = ops.load()
    pages, rows = [(n + start + 15) // 16 for n, start in lens], np.cumsum([0] + [n for n, _ in lens])
    layout = np.array([[r, n, start, p] for r, (n, start), p in zip(rows, lens, pages)], dtype=np.int32)
    cache = ops.KvCacheArgs(4096, 4096, 4096, 4096, 2, sum(pages), 16, 2, 64, 32, 1)
    step = ops.KvStepArgs(4096, 4096, 4096, 4096, None, None, layout.ctypes.data, 0, int(rows[-1]), len(lens), max(pages), 0, 0, kw.get("tiles_from", 0))
    p, q = C.byref(cache), C.byref(step)
    size = lib.kb2_seq_kv_attn_workspace(p, q, 8, 0, 0, do)
    assert size > 0
    for work, n in ((4096, size - 1), (4096, 0), (None, size), (4100, size)):
        assert lib.kb2_seq_kv_attn(p, 0, q, 4096, 0, 512, 64, 8, 1.0, 0, 0, None, 4096, do, work, n, None) == 2
