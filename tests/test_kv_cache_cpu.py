"""What the 8-bit cache and its operators refuse, without a GPU: the wrappers' checks of their arguments and the C interface's, which come before any launch."""
import ctypes as C

import numpy as np
import pytest
import torch

from krasis_b200 import seqops as ops
from krasis_b200.attention import CompactKVCache, SequenceKVState
from tests import kv_plain


def _cache(**kw):
    a = dict(num_layers=2, num_kv_heads=2, dim=64, vdim=32, device="cpu", max_pages=6, fmt="int8", page_size=16)
    a.update(kw)
    return CompactKVCache(**a)


@pytest.mark.parametrize("kw", [{"fmt": "fp8"}, {"page_size": 8}, {"page_size": 48}, {"page_size": 2048}, {"dim": 8}, {"dim": 72}, {"vdim": 272}, {"vdim": 0}, {"max_pages": 0},
                                {"num_layers": 0}, {"num_kv_heads": 0}, {"max_pages": 1 << 31}])
def test_cache_refuses(kw):
    with pytest.raises(ValueError):
        _cache(**kw)


def test_cache_pages():
    c = _cache()
    assert c.k.shape == (2, 6, 2, 16, 64) and c.v.shape == (2, 6, 2, 16, 32) and c.k_scale.shape == c.v_scale.shape == (2, 6, 2, 16)
    assert c.k.dtype == torch.int8 and _cache(fmt="e4m3").v.dtype == torch.float8_e4m3fn
    st = SequenceKVState(c)
    st.ensure_capacity(33)
    assert len(st.pages) == 3 and c.free_page_count == 3
    st.free()
    assert c.free_page_count == 6


def test_wrappers_refuse_the_cpu():
    c, tb = _cache(), ops.StepTables([([0, 0], 3, 0, [1])], "cpu")
    dt = ops.DraftTables([([0, 0], 3, 0, [1], [-1, 0])], "cpu")
    x, q = torch.zeros(2, 2, 64), torch.zeros(2, 4, 64)
    for call in (lambda: ops.kv_write(x, x[..., :32], tb, c, 0), lambda: ops.kv_read(tb, 0, 0, 1, c, 0), lambda: ops.kv_attn(q, tb, c, 0, 1.0),
                 lambda: ops.kv_tree_attn(q, dt, c, 0, 1.0), lambda: ops.kv_keep(dt, torch.zeros(1, 1, dtype=torch.int32), c)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: ops.kv_tree_attn(q, tb, c, 0, 1.0), lambda: ops.kv_attn(q, dt, c, 0, 1.0), lambda: ops.kv_keep(tb, torch.zeros(1, 1, dtype=torch.int32), c)):
        with pytest.raises(ValueError, match="DraftTables|kv_tree_attn"):
            call()


@pytest.fixture
def on_gpu(monkeypatch):
    """The wrappers' own checks: the device check is left out, and nothing may reach the library."""
    monkeypatch.setattr(ops, "_kv_call", lambda name, tb, cache, *t: (None, ops._kv_step(tb)[0], -1, {}))

    def load():
        raise AssertionError("the call should have been refused")
    monkeypatch.setattr(ops, "load", load)


def test_wrappers_refuse(on_gpu):
    c, tb = _cache(), ops.StepTables([([0, 0], 3, 0, [1])], "cpu")
    x, v, q = torch.zeros(2, 2, 64), torch.zeros(2, 2, 32), torch.zeros(2, 4, 64)
    bad = [lambda: ops.kv_write(x[:1], v, tb, c, 0), lambda: ops.kv_write(x, x, tb, c, 0), lambda: ops.kv_write(x[:, :1], v, tb, c, 0), lambda: ops.kv_write(x, v.bfloat16(), tb, c, 0),
           lambda: ops.kv_write(x.half(), v.half(), tb, c, 0), lambda: ops.kv_write(torch.zeros(2, 2, 128)[..., ::2], v, tb, c, 0), lambda: ops.kv_write(x.view(2, 128), v, tb, c, 0),
           lambda: ops.kv_read(tb, 1, 0, 1, c, 0), lambda: ops.kv_read(tb, -1, 0, 1, c, 0), lambda: ops.kv_read(tb, 0, -1, 1, c, 0), lambda: ops.kv_read(tb, 0, 0, -1, c, 0),
           lambda: ops.kv_read(tb, 0, 0, 1, c, 0, dtype=torch.float16),
           lambda: ops.kv_attn(q[:, :3], tb, c, 0, 1.0), lambda: ops.kv_attn(q[:, :0], tb, c, 0, 1.0), lambda: ops.kv_attn(q[..., :32], tb, c, 0, 1.0), lambda: ops.kv_attn(q[0], tb, c, 0, 1.0),
           lambda: ops.kv_attn(q, tb, c, 0, 1.0, window=0), lambda: ops.kv_attn(q, tb, c, 0, 1.0, window=-3), lambda: ops.kv_attn(q, tb, c, 0, 1.0, first=-1),
           lambda: ops.kv_attn(q, tb, c, 0, 1.0, sinks=torch.zeros(3)), lambda: ops.kv_attn(q, tb, c, 0, 1.0, sinks=torch.zeros(4).double()),
           lambda: ops.kv_attn(q, tb, c, 0, 1.0, out=torch.zeros(2, 4, 64)), lambda: ops.kv_attn(q, tb, c, 0, 1.0, dtype=torch.bfloat16, out=torch.zeros(2, 4, 32))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(i)


def test_drafts_refuse():
    for parents in ([-1], [-1, 1], [-1, -2], [0, 0], [-1, 0, 1]):
        with pytest.raises(ValueError):
            ops.DraftTables([([0, 0], 3, 0, [1], parents)], "cpu")
    with pytest.raises(ValueError):
        ops.DraftTables([([0, 0], 3, 0, [1], [-1, 0])], "cpu", device_buf=torch.zeros(12, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.DraftTables([([0, 0], 3, 0, [1], [-1, 0])], "cpu", device_buf=torch.zeros(10, dtype=torch.int32), draft_buf=torch.zeros(3, dtype=torch.int32))


def test_draft_tables():
    tb = ops.DraftTables([([1, 2, 3, 4], 10, 0, [0], [-1, 0, 0, 2]), ([5] * 40, 3, 1, [1], [-1] + list(range(39)))], "cpu")
    assert tb.positions[:4].tolist() == [10, 11, 11, 12] and tb.rows[:4].tolist() == [10, 11, 12, 13] and tb.words == 2
    assert tb.bits[:4, 0].tolist() == [1, 3, 5, 13] and tb.bits[:4, 1].tolist() == [0] * 4
    assert tb.positions[4:].tolist() == list(range(3, 43)) and tb.rows[4:].tolist() == list(range(3, 43))
    assert [b & 0xFFFFFFFF for b in tb.bits[43].tolist()] == [0xFFFFFFFF, 0xFF]
    assert tb.layout == ((0, 4, 10, [0]), (4, 40, 3, [1])) and tb.draft_numel == 44 * 3


# ------------------------------------------------------------------------------------------------ the C interface: refused ahead of any launch

def _structs(**kw):
    layout = np.array(kw.pop("layout", [[0, 2, 3, 1]]), dtype=np.int32)
    c = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, layers=2, pages=6, page_size=16, G=2, d=64, dv=32, fmt=1)
    s = dict(positions=4096, seq_of=4096, cu=4096, pages=4096, rows=None, bits=None, layout=layout.ctypes.data, words=0, T=2, S=len(layout), max_pages=1, replayed=0, device=0, tiles_from=0)
    step_pages = kw.pop("step_pages", 4096)
    for k, v in kw.items():
        (c if k in c else s)[k] = v
    s["pages"] = step_pages
    return ops.KvCacheArgs(**c), ops.KvStepArgs(**s), layout


@pytest.mark.parametrize("kw,code", [
    ({"k": None}, 2), ({"v_scale": None}, 2), ({"k": 4100}, 2), ({"k_scale": 4104}, 2), ({"fmt": 2}, 2), ({"fmt": -1}, 2), ({"page_size": 8}, 2), ({"page_size": 24}, 2), ({"G": 0}, 2),
    ({"d": 40}, 2), ({"dv": 512}, 2), ({"layers": 0}, 2), ({"positions": None}, 2), ({"cu": None}, 2), ({"step_pages": None}, 2), ({"layout": [[0, 2, 15, 1]]}, 4),
    ({"layout": [[0, 1, 0, 1], [1, 1, 0, 0]]}, 4), ({"layout": [[0, 2, 2147483647, 1]]}, 4), ({"S": 0}, 2), ({"T": -1}, 2), ({"max_pages": 0}, 2), ({"bits": 4096, "words": 1}, 2),
    ({"bits": 4096, "words": 0, "rows": 4096}, 2), ({"pages": 1 << 30}, 2),
    ({"bits": 4096, "words": 1, "rows": 4096, "T": 33, "layout": [[0, 33, 3, 3]], "max_pages": 3}, 2),
])
def test_interface_refuses(kw, code):
    lib = ops.load()
    c, s, keep = _structs(**kw)
    p, q = C.byref(c), C.byref(s)
    assert lib.kb2_seq_kv_write(p, 0, q, 4096, 128, 64, 4096, 64, 32, 0, None) == code
    assert lib.kb2_seq_kv_read(p, 0, q, 0, 0, 1, 4096, 4096, 0, None) == code
    assert lib.kb2_seq_kv_attn(p, 0, q, 4096, 0, 256, 64, 4, 1.0, 0, 0, None, 4096, 0, None, 0, None) == code
    assert lib.kb2_seq_kv_keep(p, q, 4096, 1, None) == code


def test_interface_refuses_arguments():
    lib = ops.load()
    c, s, keep = _structs()
    p, q = C.byref(c), C.byref(s)
    assert lib.kb2_seq_kv_write(p, 2, q, 4096, 128, 64, 4096, 64, 32, 0, None) == 4 and lib.kb2_seq_kv_write(p, -1, q, 4096, 128, 64, 4096, 64, 32, 0, None) == 4
    assert lib.kb2_seq_kv_write(p, 0, q, None, 128, 64, 4096, 64, 32, 0, None) == 2 and lib.kb2_seq_kv_write(p, 0, q, 4096, 128, 64, 4096, 64, 32, 2, None) == 2
    for s_, first, count, code in ((1, 0, 1, 2), (-1, 0, 1, 2), (0, -1, 1, 2), (0, 0, -1, 2), (0, 0, 17, 4), (0, 2147483647, 2147483647, 4)):
        assert lib.kb2_seq_kv_read(p, 0, q, s_, first, count, 4096, 4096, 0, None) == code
    assert lib.kb2_seq_kv_read(p, 0, q, 0, 0, 1, 4100, 4096, 0, None) == 2
    for H, window, first, dq, do in ((3, 0, 0, 0, 0), (1, 0, 0, 0, 0), (4, -1, 0, 0, 0), (4, 0, -1, 0, 0), (4, 0, 0, 2, 0), (4, 0, 0, 0, -1)):
        assert lib.kb2_seq_kv_attn(p, 0, q, 4096, dq, 256, 64, H, 1.0, window, first, None, 4096, do, None, 0, None) == 2
    for scale in (float("nan"), float("inf"), float("-inf")):
        assert lib.kb2_seq_kv_attn(p, 0, q, 4096, 0, 256, 64, 4, scale, 0, 0, None, 4096, 0, None, 0, None) == 2
    assert lib.kb2_seq_kv_keep(p, q, 4096, 513, None) == 2 and lib.kb2_seq_kv_keep(p, q, 4096, -1, None) == 2 and lib.kb2_seq_kv_keep(p, q, None, 1, None) == 2
    big, layout = 200000, [[0, 1, 199999, 12500]]
    c, s, keep = _structs(pages=12500, max_pages=12500, layout=layout, T=1)
    size = lib.kb2_seq_kv_attn_workspace(C.byref(c), C.byref(s), 4, 0, 0, 0)
    assert size > 0 and lib.kb2_seq_kv_attn(C.byref(c), 0, C.byref(s), 4096, 0, 256, 64, 4, 1.0, 0, 0, None, 4096, 0, 4096, size - 1, None) in (2, 3)
    assert big == layout[0][2] + 1


# ------------------------------------------------------------------------------------------------ the restatement that the GPU tests compare with

def test_restatement_quantises():
    x = np.array([[0.0, 1.0, -3.5, 448.0], [0.0, 0.0, 0.0, 0.0], [449.0, 1.0, 2.0, 3.0], [1.0, float("inf"), 0.0, 0.0]], dtype=np.float32)
    c, s = kv_plain.quantised(x, "e4m3")
    assert s[:3].tolist() == [1.0, 0.0, 2.0] and np.isnan(s[3]) and c[0].tolist() == [0.0, 1.0, -3.5, 448.0] and c[2].tolist() == [224.0, 0.5, 1.0, 1.5] and not c[3].any()
    c, s = kv_plain.quantised(x, "int8")
    assert c[0].tolist() == [0.0, 0.0, -1.0, 127.0] and s[0] == np.float32(448) * np.float32(1 / 127) and np.isnan(s[3])
    got = torch.from_numpy(np.random.RandomState(0).randn(1000, 32).astype(np.float32))
    c, s = kv_plain.quantised(got.numpy(), "e4m3")
    assert np.array_equal((got / torch.from_numpy(s)[:, None]).to(torch.float8_e4m3fn).float().numpy(), c)


def test_restatement_attends():
    c = _cache(max_pages=3, fmt="int8")
    kv_plain.fill(c, torch.Generator().manual_seed(0))
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1))
    k, v = kv_plain.held(c, 1)
    out = kv_plain.attention(q, c, 1, [(3, 17, [2, 0], None)], 0.1)[0]
    rows = [(2, j) for j in range(16)] + [(0, j) for j in range(4)]
    kk, vv = (torch.stack([x[p, 1, o] for p, o in rows]) for x in (k, v))
    want = torch.nn.functional.scaled_dot_product_attention(q[2, 3][None].double(), kk, vv, scale=0.1)
    assert torch.allclose(out[2, 3], want[0])
    chain = kv_plain.attention(q, c, 1, [(3, 17, [2, 0], [-1, 0, 1])], 0.1, window=5, first=2)[0]
    assert torch.allclose(chain, kv_plain.attention(q, c, 1, [(3, 17, [2, 0], None)], 0.1, window=5, first=2)[0])
