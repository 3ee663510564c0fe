"""Activations and weights in blocks of 128 with a scale each, and products of them, against the definition in 64 bits."""

import pytest
import torch

from tests.blocks_util import B, as_blocks, plain_codes, values_of

pytestmark = pytest.mark.gpu


def rows(T, K, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(T * 31 + K + seed)
    x = torch.randn(T, K, device="cuda", generator=g)
    x[:, torch.rand(K, device="cuda", generator=g) < 0.02] *= 20
    return x.to(dtype)


def same_codes(got, x, want, a):
    """bfloat16: every code; float32: those whose quotient is not within the two roundings before the last (2^-23) of the middle of two codes."""
    got = got.double().cpu()
    if x.dtype == torch.bfloat16:
        assert torch.equal(got, want)
        return
    off = got != want
    q = (448 * x.cpu().double() / a)[off]
    middle = (got + want)[off] / 2
    assert bool(((q - middle).abs() <= 2.0 ** -23 * middle.abs()).all())


# a row's end inside a vector of 8, a block, a multiple of 16; rows inside wider ones, at an odd element
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K,front,back", [(1, 1, 0, 0), (1, 128, 0, 0), (3, 127, 0, 0), (5, 129, 0, 0), (7, 300, 8, 4), (33, 1000, 3, 0), (130, 256, 16, 16), (2, 4100, 0, 1),
                                            (1, 513, 1, 0)])
def test_rows_in_blocks(dtype, T, K, front, back):
    from rust_llm_inference_server_b200 import ops
    wide = rows(T, front + K + back, dtype)
    x = wide[:, front:front + K]
    r = ops.quantize_rows(x)
    want, scales = plain_codes(x, 1)
    assert r.shape == (T, K) and r.scales.shape == (-(-K // B), T)
    assert torch.equal(r.scales.cpu(), scales.t())
    a = torch.clamp(torch.nn.functional.pad(x.double().abs(), (0, -K % B)).unflatten(1, (-1, B)).amax(2), min=2.0 ** -100).cpu().repeat_interleave(B, 1)[:, :K]
    same_codes(r.values, x, want, a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (127, 129), (300, 260), (3, 130, 144), (2, 40, 1000)])
def test_matrices_in_blocks(dtype, shape):
    from rust_llm_inference_server_b200 import ops
    w = rows(int(torch.tensor(shape[:-1]).prod()), shape[-1], dtype, 5).reshape(shape)
    for given in (w, w.transpose(0, 1).contiguous().transpose(0, 1) if w.dim() == 3 else w):        # matrices whose rows lie among each other's
        m = ops.quantize_matrix(given)
        for got, scales, one in zip(m.values.unsqueeze(0).flatten(0, -3), m.scales.unsqueeze(0).flatten(0, -3), w.unsqueeze(0).flatten(0, -3)):
            want, want_scales = plain_codes(one, B)
            assert torch.equal(scales.cpu(), want_scales)
            a = (want_scales.double() * 448).repeat_interleave(B, 0)[:one.shape[0]].repeat_interleave(B, 1)[:, :one.shape[1]]
            if dtype == torch.bfloat16:
                assert torch.equal(got.double().cpu(), want)
            else:
                # (a is known from its scale here, to 2^-24)
                off = got.double().cpu() != want
                q, middle = (448 * one.cpu().double() / a)[off], (got.double().cpu() + want)[off] / 2
                assert bool(((q - middle).abs() <= 2.0 ** -22 * middle.abs()).all())


def test_values_that_are_none_of_the_usual():
    from rust_llm_inference_server_b200 import ops
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.zeros(8, 300, dtype=dtype, device="cuda")
        x[1, 5] = 1e-38                         # less than the least block counts as
        x[2] = 3e38                             # 448 times it is no float32
        x[2, ::2] = -1e30
        x[3, 130] = float("nan")
        x[4, 7], x[4, 8], x[4, 200] = float("inf"), 2.0, 3.0
        x[5, 299] = float("-inf")
        x[6] = 2.0 ** -126
        r = ops.quantize_rows(x)
        v, s = r.values.float().cpu(), r.scales.cpu().t()
        least = torch.tensor(2.0 ** -100).div(448)
        assert bool((v[0] == 0).all()) and bool((s[0] == least).all()) and bool((v[1] == 0).all()) and bool((v[6] == 0).all())
        big = float(x[2, 1].float())
        assert bool((v[2, 1::2] == 448).all()) and bool((v[2, ::2] == 0).all()) and bool(((s[2] * 448 / big - 1).abs() < 1e-6).all())
        assert bool(s[3, 1].isnan()) and bool(v[3, 128:256].isnan().all()) and bool((v[3, :128] == 0).all()) and bool((v[3, 256:] == 0).all())
        assert bool(s[4, 0].isinf()) and bool(v[4, 7].isnan()) and float(v[4, 8]) == 0 and float(v[4, 200]) == 448
        assert bool(s[5, 2].isinf()) and bool(v[5, 299].isnan())
        w = rows(40, 300, torch.bfloat16, 3)
        m = ops.quantize_matrix(w)
        y = ops.linear_blocks(x, m, torch.float32)
        assert bool(y[3:6].isnan().all()) and bool(y[[0, 1, 6]].abs().max() < 1e-28) and bool((y[0] == 0).all())
        # row 2: sums of hundreds of products of 3e38 and 1 leave float32's range; where no block's and no sum of the first blocks' does, the result is finite
        parts = [(values_of(r.values, r.scales.t(), 1)[2:3, k:k + B] @ values_of(m.values, m.scales, B)[:, k:k + B].t())[0] for k in range(0, 300, B)]
        reach = torch.stack(parts + [sum(parts[:i + 1]) for i in range(len(parts))]).abs().max(0).values
        assert bool(y[2][reach < 3.4e38].isfinite().all()) and not bool(y[2][sum(parts).abs() > 3.5e38].isfinite().any())
        same = ops.linear_blocks(r, m, torch.float32)
        assert torch.equal(y[[0, 1, 2, 6, 7]], same[[0, 1, 2, 6, 7]]) and bool(same[3:6].isnan().all())


def close(y, r, m, out_dtype):
    """A block's products are exact and its sum is off by less than a unit (2^-23) for each of the four steps of 32 that an accumulator may truncate at; the
    scales' product, the product with it and the sums over blocks (in any order) by half a unit each; then one rounding to the result's type."""
    x, w = values_of(r.values, r.scales.t(), 1), values_of(m.values, m.scales, B)
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    K = x.shape[1]
    bound = (6 + K / 256) * 2.0 ** -23 * size
    half = torch.finfo(out_dtype).eps / 2
    bound = bound + half * (want.abs() + bound) + 1e-38
    assert y.dtype == out_dtype and bool(((y.double() - want).abs() <= bound).all())


SIZES = [(1, 1, 1), (1, 128, 128), (3, 40, 130), (8, 2048, 2048), (8, 1000, 4100), (16, 130, 1000), (17, 300, 513), (33, 257, 384), (64, 4096, 256), (65, 128, 1280), (100, 1, 700),
         (128, 640, 1024), (129, 255, 128), (200, 384, 129), (257, 513, 2048), (300, 2056, 640), (1, 20000, 256), (1000, 7, 64), (513, 1024, 15),
         (2, 2000, 300), (16, 2048, 2048), (16, 700, 1400), (4, 18000, 2000), (1, 300, 8000), (1, 37000, 300), (15, 260, 90),          # put into blocks by the product
         (129, 300, 3000), (130, 4100, 4100), (2000, 257, 2500), (256, 1, 1700)]          # k in shares: 3, 2, 3 and, of 14 blocks, none


@pytest.mark.parametrize("M,N,K", SIZES)
def test_products_of_blocks(M, N, K):
    from rust_llm_inference_server_b200 import ops
    x, w = rows(M, K), 0.02 * rows(N, K, torch.bfloat16, 9)
    m, r = ops.quantize_matrix(w), ops.quantize_rows(x)
    for out_dtype in (torch.bfloat16, torch.float32):
        y = ops.linear_blocks(r, m, out_dtype)
        close(y, r, m, out_dtype)
        assert torch.equal(ops.linear_blocks(x, m, out_dtype), y)                   # the same whoever puts the rows into blocks
    assert torch.equal(ops.linear_blocks(x.float(), m, torch.float32), y) and ops.linear_blocks(x, m).dtype == torch.bfloat16
    wide = torch.zeros(M, K + 5, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:3 + K] = x
    assert torch.equal(ops.linear_blocks(wide[:, 3:3 + K], m, torch.float32), y)    # rows inside wider ones
    ops.check_device_errors()


def test_a_matrix_from_a_checkpoint():
    """Scales of any size beside codes, a sign on some, rows with room behind them that holds anything."""
    from rust_llm_inference_server_b200 import ops
    for M in (4, 40, 300):
        x, w = rows(M, 200), rows(270, 200, torch.bfloat16, 2)
        m = as_blocks(w)
        room = torch.full((270, 240), float("nan"), device="cuda").to(torch.float8_e4m3fn)
        room[:, :200] = m.values
        scales = m.scales * torch.tensor([[1.0, -3.0], [1e-20, 7.5], [1e10, 0.0]], device="cuda")
        odd = ops.BlockMatrix(room[:, :200], scales)
        r = ops.quantize_rows(x)
        close(ops.linear_blocks(r, odd, torch.float32), r, odd, torch.float32)


def test_empty_and_refused_calls():
    from rust_llm_inference_server_b200 import ops
    from rust_llm_inference_server_b200.ops import KernelError
    m = ops.quantize_matrix(rows(40, 64))
    assert ops.linear_blocks(rows(0, 64), m).shape == (0, 40) and ops.quantize_rows(rows(0, 64)).shape == (0, 64)
    codes, scales = m.values, m.scales
    for bad in (lambda: ops.linear_blocks(rows(2, 65), m), lambda: ops.linear_blocks(rows(2, 64).half(), m), lambda: ops.linear_blocks(rows(2, 64), rows(40, 64)),
                lambda: ops.linear_blocks(rows(64, 2).t(), m), lambda: ops.linear_blocks(rows(2, 64), m, torch.float16), lambda: ops.linear_blocks(rows(2, 64).cpu(), m),
                lambda: ops.quantize_rows(rows(2, 64)[0]), lambda: ops.quantize_rows(rows(64, 2).t()), lambda: ops.quantize_matrix(rows(2, 64)[0]),
                lambda: ops.BlockMatrix(codes, scales.double()), lambda: ops.BlockMatrix(codes, scales[:, :0]), lambda: ops.BlockMatrix(codes[:, 1:], scales),
                lambda: ops.BlockMatrix(codes.view(torch.uint8), scales), lambda: ops.BlockMatrix(codes.t(), scales), lambda: ops.BlockRows(codes, scales),
                lambda: ops.BlockMatrix(codes[0], scales), lambda: ops.BlockMatrix(codes, scales.cpu()),
                lambda: ops.linear_blocks(rows(2, 64), ops.quantize_matrix(rows(80, 64).view(2, 40, 64)))):
        with pytest.raises(KernelError):
            bad()
