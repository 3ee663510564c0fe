"""What the ops in blocks refuse without a device."""

import pytest
import torch

from rust_llm_inference_server_b200 import ops
from rust_llm_inference_server_b200.ops import KernelError


def test_there_is_no_cpu_path():
    x, codes = torch.zeros(4, 128), torch.zeros(4, 128).to(torch.float8_e4m3fn)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.quantize_matrix(x), lambda: ops.BlockRows(codes, torch.ones(1, 4)),
                 lambda: ops.BlockMatrix(codes, torch.ones(1, 1)), lambda: ops.linear_blocks(x, x),
                 lambda: ops.moe_layer(x.bfloat16(), x, x[None].bfloat16(), x[None].bfloat16(), 1)):
        with pytest.raises(KernelError):
            call()
