"""What the classes of values in blocks refuse (no GPU needed)."""

import pytest
import torch

from rust_llm_inference_server_b200 import ops
from rust_llm_inference_server_b200.ops import KernelError


@pytest.mark.parametrize("kind", [ops.BlockRows, ops.BlockMatrix])
@pytest.mark.parametrize("values", [None, [[0.0]], 3, torch.zeros(4), torch.zeros(2, 2, 2, 2)])
def test_codes_that_are_no_matrix(kind, values):
    with pytest.raises(KernelError):
        kind(values, torch.ones(1, 1))
