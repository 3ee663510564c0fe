"""float32 into blocks: every code is the e4m3 nearest to 448 x / a, also where the quotient lies next to the middle of two codes."""

import pytest
import torch

from tests.blocks_util import B, plain_codes

pytestmark = pytest.mark.gpu


def near_middles(rows, K, seed, size=1.0):
    """Rows whose blocks begin with their largest value a, and whose other values are the float32 next to m a / 448 for middles m of two codes, up to two units away.
    (In 64 bits the definition tells them apart: 7 x has 27 bits and m a 29, so the quotient is at least 2^-29 of it away from m, or m.)"""
    g = torch.Generator().manual_seed(seed)
    a = size * (1 + torch.rand(rows, K // B, 1, generator=g))
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middles = (codes[1:] + codes[:-1]) / 2
    m = middles[torch.randint(0, len(middles), (rows, K // B, B - 1), generator=g)]
    x = (m * a.double() / 448).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=g).int()).view(torch.float32)
    x = x * (1 - 2 * torch.randint(0, 2, x.shape, generator=g))
    return torch.cat([a, x], 2).reshape(rows, K).cuda()


@pytest.mark.parametrize("size", [1.0, 2.0 ** -99, 1e-9, 2.0 ** 101, 2.0 ** 126])
def test_codes_next_to_the_middle_of_two(size):
    from rust_llm_inference_server_b200 import ops
    x = near_middles(24, 1024, 3, size)
    want, scales = plain_codes(x, 1)
    rows = ops.quantize_rows(x)
    assert torch.equal(rows.values.double().cpu(), want) and torch.equal(rows.scales.t().cpu(), scales)
    want, scales = plain_codes(x, B)
    matrix = ops.quantize_matrix(x)
    assert torch.equal(matrix.values.double().cpu(), want) and torch.equal(matrix.scales.cpu(), scales)


def test_values_that_two_roundings_take_to_the_wrong_code():
    from rust_llm_inference_server_b200 import ops
    x = torch.zeros(3, 4, device="cuda")
    for i, (a, v) in enumerate([(1.0409735441207886, 0.0003812159120570868), (1.0165276527404785, 0.0026944789569824934), (1.9127556085586548, 0.03095419332385063)]):
        x[i] = torch.tensor([a, v, -v, 0.0])
    codes = ops.quantize_rows(x).values.float()
    assert codes[:, 1].tolist() == [0.171875, 1.125, 7.5] and torch.equal(codes[:, 2], -codes[:, 1])


@pytest.mark.parametrize("T", [1, 16, 60])
def test_products_of_float32_rows_are_those_of_their_codes(T):
    from rust_llm_inference_server_b200 import ops
    x, w = near_middles(T, 1024, 5), ops.quantize_matrix(near_middles(300, 1024, 6))
    assert torch.equal(ops.linear_blocks(x, w), ops.linear_blocks(ops.quantize_rows(x), w, torch.float32))


def test_random_float32_codes():
    from rust_llm_inference_server_b200 import ops
    x = torch.randn(2048, 2048, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    a = x.view(2048, 16, B).abs().amax(2, keepdim=True).double()
    q = 448 * x.view(2048, 16, B).double() / a
    m, _ = torch.frexp(q)
    step = torch.where(q == 0, torch.zeros_like(q), q / m / 16).clamp(min=2.0 ** -9)
    want = (torch.round(q / step) * step).view(2048, 2048)
    assert torch.equal(ops.quantize_rows(x).values.double(), want)
