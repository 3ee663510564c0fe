"""Products of blocks beside the framework's other products on another stream: both want tensor memory, and both meet in clusters."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(sum((i + 1) * s for i, s in enumerate(shape)) + seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


@pytest.mark.parametrize("rows", [2, 16, 40, 100])
@pytest.mark.parametrize("other", ["stream", "float32"])
def test_products_of_blocks_beside_other_products(rows, other):
    from rust_llm_inference_server_b200 import ops
    dtype = torch.bfloat16 if other == "stream" else torch.float32
    xs, ws = [rand(rows, 2048), rand(12, 2048, dtype=dtype)], [ops.quantize_matrix(rand(2048, 2048, scale=0.03)), rand(2048, 2048, scale=0.03, dtype=dtype)]
    calls = [lambda: ops.linear_blocks(xs[0], ws[0], torch.float32), lambda: ops.linear(xs[1], ws[1], torch.float32)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        for i, (c, s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(c())
    torch.cuda.synchronize()
    assert all(torch.equal(y, v) for g, v in zip(got, want) for y in g)
    ops.check_device_errors()
