"""The expert layer with gates far below zero: silu(g) is g exp(g) there, and a hidden value of any size beside a large second product.
Gates are exact sums of 64 products (see test_mx_grouped_edges) and a hidden value goes to one output, so what is left is silu, off by 2^-20,
three products and the weight, 2^-20 together, and what that does to a code (mx_helpers.requantized)."""
import numpy as np
import pytest

import mx_helpers as mx
from computelibrary_b200 import capi
from test_mx_grouped_edges import ONE, whole
from test_mx_moe import workspace


class Exact:
    """One expert: gates `gates` for a row of ones, up values of one, hidden value f to output f."""

    def __init__(self, gates, fmt):
        import torch
        def matrix(code):
            byte = np.full((code.shape[0], mx.blocks_of(code.shape[1], fmt)), ONE[fmt], np.uint8)
            return torch.from_numpy(mx.pack(code, capi.mx_pitch(code.shape[1]))).cuda(), torch.from_numpy(mx.tile(byte)).cuda()

        self.gate = matrix(whole(gates))
        self.up = matrix(whole(np.ones(len(gates))))
        self.down = matrix((2 * np.eye(len(gates))).astype(np.uint8))


def stored_hidden(gates, fmt, exponent):
    """(hidden values as they are stored, bound of what their error changes)."""
    one = mx.values(*mx.quantize(np.ones((1, 64)), fmt), fmt)[0, 0]  # what a row of ones is stored as
    g = gates * one
    h = (g / (1 + np.exp(-g)) * one * 2.0 ** 100)[None]
    return mx.requantized(h, 2.0 ** -19 * np.abs(h), fmt, exponent)


HIDDEN = [(capi.MXFP4, 0), (capi.NVFP4, -40), (capi.NVFP4, -30)]  # the second saturates


@pytest.mark.parametrize("fmt,exponent", HIDDEN)
def test_hidden_values_are_not_zero(fmt, exponent):
    """What the test below compares with can tell them from 0."""
    gates = np.repeat([-86.0, -87.5, -89.0, -92.0], 16) - np.arange(64) % 4 / 2
    y, tol = stored_hidden(gates, fmt, exponent)
    assert (np.abs(y) > 2 * tol).sum() >= 40


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,exponent", HIDDEN)
@pytest.mark.parametrize("tokens", [1, 5, 128])
def test_gates_far_below_zero(ctx, fmt, exponent, tokens):
    import torch
    gates = np.repeat([-86.0, -87.5, -89.0, -92.0], 16) - np.arange(64) % 4 / 2  # near enough in a block for codes other than 0
    layer = Exact(gates, fmt)
    x = torch.ones((tokens, 64), dtype=torch.bfloat16, device="cuda")
    logits = torch.zeros((tokens, 1), device="cuda")
    d = capi.make_mx_moe_desc(tokens, 64, 64, 1, 1, fmt, capi.BF16, up_alpha=2.0 ** 100, h_exponent=exponent)
    out = torch.full((tokens, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.mx_moe(d, x, logits, layer.gate, layer.up, layer.down, out, workspace(d))
    ctx.sync()
    y, tol = stored_hidden(gates, fmt, exponent)
    got = out.double().cpu().numpy()
    bad = ~(np.abs(got - y) <= tol + 2.0 ** -8 * (np.abs(y) + tol))
    assert not bad.any(), f"{bad.sum()} of {bad.size} off: {got[bad][:3]} for {np.broadcast_to(y, got.shape)[bad][:3]}"
