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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [capi.F32, capi.F16, capi.BF16])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(7, 8, 3), (300, 200, 6)])
def test_route_infinite_logits(ctx, T, E, k, renormalize, dtype):
    """+infinity is the largest logit there is, and infinity over infinity is NaN: so are all weights of its token, and of no other."""
    import torch
    rng = np.random.default_rng(T)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    clean = logits.copy()
    logits[2, 5] = logits[2, 3] = logits[T - 1, E - 1] = np.inf
    ids, w, slots, groups = check_route(ctx, clean, k, dtype, renormalize)
    want = ids.clone(), w.clone()
    x = torch.from_numpy(logits).to({capi.F32: torch.float32, capi.F16: torch.float16, capi.BF16: torch.bfloat16}[dtype]).cuda()
    d = capi.make_moe_route_desc(T, E, k, dtype, renormalize)
    ws = torch.zeros(capi.moe_route_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    ctx.moe_route(d, x, ids, w, slots, groups, ws)
    ctx.sync()
    assert ids[2, :2].tolist() == [3, 5] and ids[T - 1, 0] == E - 1
    others = [t for t in range(T) if t not in (2, T - 1)]
    assert torch.equal(ids[others], want[0][others]) and torch.equal(w[others], want[1][others])
    assert torch.isnan(w[2]).all() and torch.isnan(w[T - 1]).all()
    assert sorted(slots[:T].flatten().tolist()) == sorted(r for s, c in groups[:E].tolist() for r in range(s, s + c)) and groups[:E, 1].sum() == T * k


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [capi.MXFP4, capi.NVFP4])
@pytest.mark.parametrize("T,cols", [(30, 256), (600, 1024), (30, 131)])
def test_group_the_same_row_twice_in_a_token(ctx, T, cols, fmt):
    """A token whose choices name a row twice writes it once or twice alike; rows that are no longer named are not written at all."""
    import torch
    d, src, slots, packed, tiles = check_group(ctx, T, 4, cols, fmt, capi.BF16, missing=0.0)
    want, want_tiles = packed.clone(), tiles.clone()
    slots[2:, 3] = slots[2:, 1]
    packed.fill_(0x5A)
    tiles.fill_(0x5A)
    ctx.mx_quantize_grouped(d, src, slots, packed, tiles)
    ctx.sync()
    rows = d.rows
    named = torch.zeros(rows, dtype=torch.bool)
    inside = slots[(slots >= 0) & (slots < rows)].long().cpu()
    named[inside] = True
    named = named.cuda()
    used = (cols + 1) // 2
    assert torch.equal(packed[named, :used], want[named, :used])
    assert (packed[~named] == 0x5A).all() and (packed[:, used:] == 0x5A).all()
    import mx_helpers as mx
    words = -(-mx.blocks_of(cols, fmt) // 4) * 4
    got, old = (mx.untile(t.cpu().numpy(), rows, words) for t in (tiles, want_tiles))
    keep = named.cpu().numpy()
    assert (got[keep] == old[keep]).all() and (got[~keep] == 0x5A).all()
