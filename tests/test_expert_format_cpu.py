"""Asking for experts in 8-bit floating point: which designs take it, and what is said ahead of reading a checkpoint."""
import json

import pytest


def _dir(tmp_path, cfg):
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    return str(tmp_path)


@pytest.mark.parametrize("cfg", [{"architecture": a} for a in ("Vofelix", "Gurozen", "Zaronex", "Kugalorn", "Kivurax")]
                         + [{"model_type": "qwen3_moe"}, {"text_config": {"model_type": "qwen3_5_moe_text"}}])
def test_designs_that_do_not_take_the_format_refuse_it(tmp_path, monkeypatch, cfg):
    """By load_model itself, ahead of building, importing or reading anything."""
    from krasis_b200 import build, registry
    for name in ("build", "build_seq"):
        monkeypatch.setattr(build, name, lambda: pytest.fail("built"))
    with pytest.raises(ValueError, match="does not hold its experts in e4m3"):
        registry.load_model(_dir(tmp_path, cfg), expert_format="e4m3")


def test_a_design_from_outside_takes_the_word_itself(tmp_path, monkeypatch):
    from krasis_b200 import registry
    monkeypatch.setattr(registry, "_REGISTRY", dict(registry._REGISTRY))
    registry.register("Elsewhere", lambda d, dtype, device, **kw: kw)
    assert registry.load_model(_dir(tmp_path, {"architecture": "Elsewhere"}), expert_format="e4m3") == {"expert_format": "e4m3"}


@pytest.mark.parametrize("kw", [{}, {"expert_format": None}])
def test_designs_load_without_the_word_as_before(tmp_path, monkeypatch, kw):
    from krasis_b200 import registry
    seen = []
    monkeypatch.setitem(registry._REGISTRY, "Kivurax", lambda d, dtype, device, **k: seen.append(k))
    registry.load_model(_dir(tmp_path, {"architecture": "Kivurax"}), **kw)
    assert seen == [kw]


@pytest.mark.parametrize("kw,want", [({}, ["seq"]), ({"expert_format": "e4m3"}, ["seq", "core"])])
def test_the_libraries_that_a_load_needs_are_built_ahead_of_it(tmp_path, monkeypatch, kw, want):
    """Experts in 8 bits run on the core library, which a design of the sequence library does not build otherwise."""
    from krasis_b200 import build, megolorn, registry
    done = []
    monkeypatch.setattr(build, "build_seq", lambda: done.append("seq"))
    monkeypatch.setattr(build, "build", lambda: done.append("core"))
    monkeypatch.setattr(megolorn.MegolornModel, "from_pretrained", classmethod(lambda cls, *a, **k: done.append("read")))
    layers = [{"type": "attention", "mixer": {"heads": 2, "kv_heads": 1, "dim": 16, "vdim": 16, "scale": 0.25},
               "mlp": {"kind": "moe", "expert": {"ff": 128}, "router": {"experts": 4, "top": 2}}}]
    registry.load_model(_dir(tmp_path, {"architecture": "Megolorn", "vocab": 50, "width": 32, "norm": {"eps": 1e-5}, "layers": layers}), **kw)
    assert done == want + ["read"]


def _megolorn(experts=4, identity=0, ff=128, width=32):
    router = {"experts": experts, "identity": identity, "top": 2}
    layers = [{"type": "attention", "mixer": {"heads": 2, "kv_heads": 1, "dim": 16, "vdim": 16, "scale": 0.25}, "mlp": mlp}
              for mlp in (None, {"ff": 56, "limit": 0.5}, {"kind": "moe", "expert": {"ff": ff}, "router": router})]
    return {"architecture": "Megolorn", "vocab": 50, "width": width, "norm": {"eps": 1e-5}, "layers": layers}


UNFIT = [({"identity": 1}, "identity"), ({"experts": 1025}, "1024"), ({"experts": 0, "identity": 0}, "1024"), ({"ff": 120}, "inner width 120"), ({"width": 24}, "width 24")]


@pytest.mark.parametrize("sizes,said", UNFIT)
def test_sizes_that_do_not_fit_are_named_ahead_of_reading(tmp_path, monkeypatch, capsys, sizes, said):
    """By load_model, the class and the command line, from config.json alone."""
    from krasis_b200 import build, loader, megolorn, registry
    from krasis_b200.__main__ import main
    for where, name in ((build, "build"), (build, "build_seq"), (loader, "read_named_tensors")):
        monkeypatch.setattr(where, name, lambda *a: pytest.fail("built or read"))
    d = _dir(tmp_path, _megolorn(**sizes))
    for load in (registry.load_model, megolorn.MegolornModel.from_pretrained):
        with pytest.raises(ValueError, match=said):
            load(d, expert_format="e4m3")
    assert main(["score", "--model", d, "--prompt-ids", "1,2", "--expert-format", "e4m3"]) == 3
    assert said in capsys.readouterr().err


def test_formats_that_there_are_not(tmp_path):
    from krasis_b200 import registry
    from krasis_b200.megolorn import MegolornConfig
    with pytest.raises(ValueError, match="expert format 'e5m2'"):
        registry.load_model(_dir(tmp_path, _megolorn()), expert_format="e5m2")
    dense = _megolorn()
    dense["layers"] = dense["layers"][:2]
    for cfg in (_megolorn(), _megolorn(identity=2, ff=24), dense):
        MegolornConfig.from_dict(cfg).check_expert_format(None)
        with pytest.raises(ValueError):
            MegolornConfig.from_dict(cfg).check_expert_format("int4")
    for cfg in (_megolorn(), _megolorn(experts=1024, width=16, ff=256), dense):
        MegolornConfig.from_dict(cfg).check_expert_format("e4m3")
