"""The routed layer with infinite numbers in it: a sum that is infinite is that, and no NaN."""

import pytest
import torch

from tests.blocks_util import B

pytestmark = pytest.mark.gpu


def layer(x, up, down, blocks, **more):
    """Two experts, of which every token takes the first with weight 1, and units max(gate, 0) lin."""
    from rust_llm_inference_server_b200 import ops
    W = x.shape[1]
    router = torch.zeros(2, W, device="cuda")
    if blocks:
        def stored(m):
            m = torch.stack([m, m.sign()])
            scales = m.unflatten(2, (-1, m.shape[2])).abs().amax((1, 2, 3)).clamp(min=2.0 ** -90) / 4          # the largest code is 4
            return ops.BlockMatrix((m / scales[:, None, None]).cuda().to(torch.float8_e4m3fn), scales[:, None, None].expand(-1, -(-m.shape[1] // B), -(-m.shape[2] // B)).contiguous().cuda())
    else:
        stored = lambda m: torch.stack([m, m.sign()]).bfloat16().cuda()
    return ops.moe_layer(x.bfloat16().cuda(), router, stored(up), stored(down), 1, scoring="softmax_chosen", slope=float("inf"), **more).float().cpu()


def inputs(T, W, I, first, second, third):
    """Feature 5's gate is x[0] and its linear branch x[1] + x[2]; the others' are the small x[3] and x[4]."""
    x = torch.zeros(T, W)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3], x[:, 4] = first, second, third, 2.0, 3.0
    up = torch.zeros(2 * I, W)
    up[:I, 3], up[I:, 4] = 1, 1
    up[5], up[I + 5] = 0, 0
    up[5, 0], up[I + 5, 1], up[I + 5, 2] = 1, 1, 1
    return x, up


@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("T", [1, 6, 14])
def test_an_infinite_gated_result(T, blocks):
    W, I = 48, 144
    x, up = inputs(T, W, I, 2.0 ** 100, 2.0 ** 100, 0.0)
    down = torch.ones(W, I)
    down[::2, 5] = -1
    y = layer(x, up, down, blocks)
    assert bool((y[:, 1::2] == float("inf")).all()) and bool((y[:, ::2] == float("-inf")).all())
    x[:, 1] = -x[:, 1]
    assert bool((layer(x, up, down, blocks) == -y).all())


@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("T", [1, 6, 14])
def test_a_gated_result_beyond_the_largest_bfloat16(T, blocks):
    """2^127 (2 - 2^-9) is a float32, and nearest to it is the bfloat16 infinity.  (In blocks the second product's largest code is 4, four times its weight's.)"""
    W, I = 48, 144
    x, up = inputs(T, W, I, 2.0 ** 64, 2.0 ** 63 * 255 / 128, 2.0 ** 63 * (1 / 128 - 2.0 ** -9))
    down = torch.zeros(W, I)
    down[:, 5] = 2.0 ** -10
    down[1::2, 5] = -2.0 ** -20
    y = layer(x, up, down, blocks)
    want = (down[:, 5].double() * 2.0 ** 127 * (2 - 2.0 ** -9)).bfloat16().float()
    assert torch.equal(y, want.expand(T, W))


@pytest.mark.parametrize("T", [1, 6, 14])
def test_an_infinite_weight(T):
    """Of the second product, times numbers of either sign that need both of their parts."""
    W, I = 48, 144
    g = torch.Generator().manual_seed(T)
    for at in (0, 17, 130):
        x, up = torch.rand(T, W, generator=g) + 0.5, torch.rand(2 * I, W, generator=g) + 0.5
        down = torch.rand(W, I, generator=g) - 0.5
        down[3, at], down[40, at] = float("inf"), float("-inf")
        y = layer(x, up, down, False)
        assert bool((y[:, 3] == float("inf")).all()) and bool((y[:, 40] == float("-inf")).all()) and bool(y[:, :3].isfinite().all()) and bool(y[:, 41:].isfinite().all())
        assert bool((layer(-x, torch.cat([-up[:I], up[I:]]), down, False)[:, 3] == float("-inf")).all())


@pytest.mark.parametrize("T", [1, 6, 14])
def test_an_infinite_weight_at_its_row_s_end(T):
    """Rows that end inside a chunk of 128: nothing past the end takes part."""
    W, I = 200, 144
    g = torch.Generator().manual_seed(T)
    x, up = torch.rand(T, W, generator=g) + 0.5, torch.rand(2 * I, W, generator=g) + 0.5
    down = torch.rand(W, I, generator=g) - 0.5
    for at in (I - 8, I - 1):
        bad = down.clone()
        bad[3, at], bad[199, at] = float("inf"), float("-inf")
        y = layer(x, up, bad, False)
        assert bool((y[:, 3] == float("inf")).all()) and bool((y[:, 199] == float("-inf")).all()) and bool(y[:, :3].isfinite().all()) and bool(y[:, 4:199].isfinite().all())
    for row in (20, I + 20):                # a gate's, a linear branch's
        for at in (W - 8, W - 1):
            bad = up.clone()
            bad[row, at] = float("inf")
            y, sign = layer(x, bad, down, False), down[:, 20].sign()
            assert torch.equal(y, (sign * float("inf")).expand(T, W))
