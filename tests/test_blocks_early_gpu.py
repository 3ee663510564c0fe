"""`early`, the caller's word that no kernel in flight writes a weight, reaches the product whoever puts its rows into blocks."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,given", [(1, False), (8, False), (8, True), (100, True), (200, True)])
def test_a_product_is_told_that_its_weight_is_loaded(monkeypatch, T, given):
    from rust_llm_inference_server_b200 import ops
    from rust_llm_inference_server_b200.ops import blocks
    x, w = torch.randn(T, 512, device="cuda"), ops.quantize_matrix(torch.randn(640, 512, device="cuda"))
    rows = ops.quantize_rows(x) if given else x
    want, told, kernels = ops.linear_blocks(rows, w), [], blocks.lib()

    class Listening:
        def __getattr__(self, name):
            call = getattr(kernels, name)
            if name not in ("rlis_blocks_gemm", "rlis_blocks_gemm_rows"):
                return call
            return lambda *args: (told.append(args[-2]), call(*args))[1]

    monkeypatch.setattr(blocks, "lib", Listening)
    assert torch.equal(ops.linear_blocks(rows, w, want.dtype, early=True), want) and torch.equal(ops.linear_blocks(rows, w, want.dtype), want)
    assert told == [1, 0]


@pytest.mark.parametrize("T", [1, 8, 40])
def test_plain_rows_that_the_kernel_before_writes(T):
    """Only the weight may be read early."""
    from rust_llm_inference_server_b200 import ops
    w = ops.quantize_matrix(torch.randn(2048, 1024, device="cuda"))
    xs = [torch.randn(T, 1024, device="cuda") for _ in range(4)]
    want = [ops.linear_blocks(x, w, torch.float32) for x in xs]
    x = torch.empty(T, 1024, device="cuda")
    torch.cuda.synchronize()
    got = []
    for i in range(40):
        x.copy_(xs[i % 4])
        got.append(ops.linear_blocks(x, w, torch.float32, early=True))
    first = ops.linear_blocks(ops.linear_blocks(xs[0], w, early=True)[:, :1024], w, early=True)
    again = ops.linear_blocks(ops.linear_blocks(xs[0], w)[:, :1024], w)
    assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(got)) and torch.equal(first, again)
    ops.check_device_errors()


@pytest.mark.parametrize("N,K", [(2048, 2048), (700, 4100), (300, 14336)])
def test_a_row_s_bits_do_not_depend_on_the_rows_beside_it(N, K):
    """Up to 64 rows, whoever puts them into blocks."""
    from rust_llm_inference_server_b200 import ops
    x, w = torch.randn(64, K, device="cuda").bfloat16(), ops.quantize_matrix(torch.randn(N, K, device="cuda"))
    whole = ops.linear_blocks(x, w, torch.float32)
    for first, last in ((0, 1), (5, 6), (0, 2), (3, 19), (60, 64), (10, 42), (0, 63)):
        assert torch.equal(ops.linear_blocks(x[first:last], w, torch.float32), whole[first:last])
        assert torch.equal(ops.linear_blocks(ops.quantize_rows(x[first:last]), w, torch.float32), whole[first:last])
