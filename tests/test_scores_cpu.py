"""Which tokens the scheduler runs to score texts, with a stand-in model on the CPU."""
import pytest

from tests.test_logprobs_serving_cpu import sched  # noqa: F401


@pytest.mark.parametrize("n,portion,sizes", [(0, 4, []), (1, 4, []), (2, 4, [1]), (4, 4, [3]), (5, 4, [4]), (6, 4, [4, 1]), (9, 4, [4, 4]), (3, 1, [1, 1]), (7, 100, [6])])
def test_no_token_is_run_that_nothing_follows(sched, n, portion, sizes):  # noqa: F811
    text = [(3 * i) % 13 for i in range(n)]
    got = sched.score([text], step_tokens=portion)
    assert len(got[0]) == max(n - 1, 0)
    assert [tb.tokens.numel() for tb in sched.model.steps] == sizes
    assert [t for tb in sched.model.steps for t in tb.tokens.tolist()] == text[:-1]
    assert not sched.live and sched.kv_cache.free_page_count == 16


def test_texts_of_one_token_beside_live_requests(sched):  # noqa: F811
    for r in range(3):
        sched.step([(r, [1, 2], [])])
    assert sched.score([[5], []]) == [[], []]
    with pytest.raises(RuntimeError, match="does not fit"):
        sched.score([[5, 6]])
    assert len(sched.live) == 3
