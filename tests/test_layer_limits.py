"""Sizes at the ends of the C entry points' argument types, without a GPU: refused by
arithmetic that holds them, before any launch."""

import pytest

from calibration_free_moe.reader import _ext
from tests.test_layer_refusals import call_experts, call_route, refused

INT32_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("tokens", [INT32_MAX, INT32_MAX - 14, INT32_MAX - 15])
@pytest.mark.parametrize("experts", [8, 1024])
def test_route_refuses_the_largest_token_counts(tokens, experts):
    refused(call_route(experts=experts, tokens=tokens), "too many tokens")
    tiles = (experts + 15) // 16
    assert _ext.library().cfmoe_route_scratch_bytes(tokens, experts) == 4 * tokens * (experts + tiles)


def test_routed_experts_refuses_the_largest_token_counts():
    for top_k in (1, 2, 64):
        refused(call_experts(tokens=INT32_MAX, top_k=top_k), "8192")
