"""Places in a kernel's shared memory: what lives from the kernel's start to its end under two names must not lie in one place."""
import re

from tests.test_pdl import _bodies


def _places(body):
    """{place: names} of the pointers that a kernel's outermost block declares, where they begin."""
    depth, flat = 0, []
    for c in body:                                         # what stands in inner blocks lives shorter
        depth += {"{": 1, "}": -1}.get(c, 0)
        flat.append(c if depth == 1 and c != "}" else ";" if depth == 1 else " ")
    out = {}
    for statement in "".join(flat).split(";"):
        if re.match(r"\s*(?:const\s+)?[\w:]+\s*\*", statement):
            for name, place in re.findall(r"\*\s*(\w+)\s*=\s*([^,]+(?:\([^)]*\)[^,]*)*)", statement):
                out.setdefault(re.sub(r"\s+", "", place), []).append(name)
    return out


def test_no_two_names_for_one_place():
    seen = 0
    for kernel, (_, body) in _bodies().items():
        for place, names in _places(body).items():
            seen += 1
            assert len(names) == 1, (kernel, place, names)
    assert seen > 100


def test_two_names_are_found():
    body = "{ uint32_t* have = reinterpret_cast<uint32_t*>(refs + 4); uint32_t* gone = have + 3; if (x) { int* a = have + 5; } uint32_t *tmem_at = have + 3, *b = have + 5; }"
    assert _places(body)["have+3"] == ["gone", "tmem_at"] and _places(body)["have+5"] == ["b"]
