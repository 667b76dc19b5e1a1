"""Loads through a __restrict__ pointer may move ahead of a programmatic launch's wait, so each such parameter goes through the wait (csrc/pdl.cuh)."""
import re

from tests.test_pdl import _bodies, _launched


def _left_out(params, body):
    through = re.search(r"pdl_(?:enter|enter_global|wait)\(([^;]*)\);", body).group(1)
    return [p for p in re.findall(r"__restrict__\s+(\w+)", params) if not re.search(r"\b%s\b" % p, through)]


def test_restricted_pointers_go_through_the_wait():
    bodies, seen = _bodies(), 0
    for kernel in sorted(_launched()):
        params, body = bodies[kernel]
        seen += len(re.findall("__restrict__", params))
        assert not _left_out(params, body), (kernel, _left_out(params, body))
    assert seen > 100


def test_one_that_does_not_is_found():
    assert _left_out("KvLayer c, const int* __restrict__ path, float* __restrict__ o", "{ kb2::pdl_enter(o); }") == ["path"]
