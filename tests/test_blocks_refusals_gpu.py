"""Refusals of the ops in blocks that name what they want."""

import pytest
import torch

from tests.test_moe_layer_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 2, 16])
def test_rows_of_the_layer_that_start_anywhere(T):
    from rust_llm_inference_server_b200 import ops
    from rust_llm_inference_server_b200.ops import KernelError
    m = make(T, 128, 32, 4)
    wide = torch.zeros(T, 144, dtype=torch.bfloat16, device="cuda")
    for front in (1, 4, 7):
        with pytest.raises(KernelError, match="16 bytes"):
            ops.moe_layer(wide[:, front:front + 128], m["router"], m["up"], m["down"], 2)
    uneven = torch.zeros(T, 132, dtype=torch.bfloat16, device="cuda")[:, :128]
    if T > 1:
        with pytest.raises(KernelError, match="16 bytes"):
            ops.moe_layer(uneven, m["router"], m["up"], m["down"], 2)
    else:
        assert bool((ops.moe_layer(uneven, m["router"], m["up"], m["down"], 2) == 0).all())
    wide[:, 8:136] = m["x"]
    assert torch.equal(ops.moe_layer(wide[:, 8:136], m["router"], m["up"], m["down"], 2), ops.moe_layer(m["x"], m["router"], m["up"], m["down"], 2))


def test_what_is_no_tensor():
    from rust_llm_inference_server_b200 import ops
    from rust_llm_inference_server_b200.ops import KernelError
    m = make(2, 128, 32, 4, 32)
    layer = lambda **c: ops.moe_layer(m["x"], c.pop("router", m["router"]), m["up"], m["down"], 2, **c)
    layer()
    for call in (lambda: layer(router=[0.0] * 4), lambda: layer(correction=[0.0] * 4), lambda: layer(router_bias=0.5), lambda: layer(out=[]), lambda: layer(shared=([], m["shared_down"])),
                 lambda: ops.linear_blocks([[1.0]], ops.quantize_matrix(m["router"])), lambda: ops.linear_blocks(m["x"], None), lambda: ops.quantize_matrix([1.0])):
        with pytest.raises(KernelError):
            call()
