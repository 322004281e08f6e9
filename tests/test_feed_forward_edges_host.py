"""Contracts of the feed-forward operators that need no GPU."""
import math

import torch

from oracle import feed_forward as O


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
