"""Contracts of the feed-forward operators that need no GPU."""
import math

import pytest
import torch

from flashnn_b200 import _lib
from oracle import feed_forward as O


@pytest.fixture(scope="module")
def lib():
    from flashnn_b200 import build
    build.build()
    return _lib.lib()


def test_ranges_of_experts_that_pass_32_bits_are_refused(lib):
    """Experts 2^31 - 4 .. 2^31 would wrap to -2^31, which is a number that a choice can have."""
    def sort(first, e):
        return lib.fnn_moe_sort(None, 8, e, first, 16, None, lib.fnn_moe_sort_slots(8, e, 16), None, None, None)

    def combine(first, e, ids=16):
        return lib.fnn_moe_combine(None, _lib.BF16, 64, 32, 4, 2, 32, None, ids, e, first, None, 0, None, 32, None)
    for call in (sort, combine):
        assert call(2 ** 31 - 4, 5) == 3 and b"32 bits" in lib.fnn_last_error_string()
        assert call(2 ** 31 - 1, 2) == 3 and call(2 ** 63 - 1, 4) == 3 and call(-2 ** 31 - 1, 4) == 3
        assert call(2 ** 31 - 4, 4) == 1 and call(-2 ** 31, 4) == 1  # (as far as the missing tensors)
    assert combine(5, 2 ** 31 - 1) == 3 and combine(0, 2 ** 31 - 1) == 1
    assert combine(5, 2 ** 31 - 1, ids=None) == 1  # without ids the range says nothing


def test_with_a_bias_only_a_bias_of_minus_infinity_takes_an_expert_out():
    """The definition's own words: key = score + bias, so a score of 0 competes with its bias."""
    x = torch.zeros(1, 24)
    x[0, 0] = -math.inf
    bias = torch.zeros(24)
    bias[0] = 0.2
    for scoring, group in (("softmax", {}), ("softmax", dict(num_groups=3, topk_groups=2, group_score="top2"))):
        w, ids = O.route(x, 2, bias, scoring=scoring, **group)
        assert ids.tolist() == [[0, 1]] and w.tolist() == [[0.0, 1.0]]
    assert 0 not in O.route(x, 2)[1] and 0 not in O.route(x, 2, scoring="sigmoid")[1]
    bias[0] = -math.inf
    for scoring in ("softmax", "sigmoid"):
        for logits in (x, torch.full((1, 24), 3.0)):
            assert 0 not in O.route(logits, 2, bias, scoring=scoring)[1]
