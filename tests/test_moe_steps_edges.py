"""The steps of an expert layer at the edges: as many tokens as 32 bits count, infinite logits, rows that are written again."""
import numpy as np
import pytest

from computelibrary_b200 import capi
from test_moe_steps import check_group, check_route

MOST = 2 ** 31 - 1 - 1024 - 128  # tokens of a gate with one expert


@pytest.mark.parametrize("tokens", [MOST, MOST - 1, 2 ** 31 - 2 ** 23, 2 ** 30, 2 ** 30 + 1, 4737, 33])
def test_workspace_of_the_largest_gates(tokens):
    """At most 256 chunks, whatever the number of tokens."""
    d = capi.make_moe_route_desc(tokens, 1, 1, capi.BF16)
    assert capi.moe_route_validate(d)[0] == 0
    assert 4 <= capi.moe_route_workspace_bytes(d) <= 256 * 4


def test_one_token_more_is_refused():
    assert capi.moe_route_validate(capi.make_moe_route_desc(MOST + 1, 1, 1, capi.BF16))[0] == capi.INVALID_ARGUMENT


@pytest.mark.gpu
def test_route_as_many_tokens_as_32_bits_count(ctx):
    import torch
    logits = torch.zeros(MOST, dtype=torch.bfloat16, device="cuda")
    logits[::3] = float("nan")  # nothing to choose
    logits[-1] = 1.0
    d = capi.make_moe_route_desc(MOST, 1, 1, capi.BF16)
    ids, slots = (torch.full((MOST,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    w = torch.full((MOST,), 77.0, device="cuda")
    groups = torch.full((1, 2), 77, dtype=torch.int32, device="cuda")
    ws = torch.full((capi.moe_route_workspace_bytes(d),), 255, dtype=torch.uint8, device="cuda")
    ctx.moe_route(d, logits, ids, w, slots, groups, ws)
    ctx.sync()
    last, chosen = MOST - 1, 0
    for start in range(0, MOST, 2 ** 28):
        rows = slice(start, min(start + 2 ** 28, MOST))
        has = ~torch.isnan(logits[rows])
        assert torch.equal(ids[rows], has.int() - 1) and torch.equal(w[rows], has.float())
        place = torch.cumsum(has, 0, dtype=torch.int32) - 1 + chosen
        assert torch.equal(slots[rows], torch.where(has, place, -1))
        chosen += int(has.sum())
    assert groups.tolist() == [[0, chosen]] and ids[last] == 0
