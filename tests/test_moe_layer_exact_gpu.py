"""The routed layer where every number of it is a small whole number: what its parts hold in fewer bits than float32 shows as a wrong digit."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def whole_layer(T, blocks, most_x, seed):
    """One of two experts a token, its weight exactly 1, units max(gate, 0) lin.  Features in pairs of gated results h that differ by gate * x[2] alone, which is what the
    second product gives: the differences of neighbours.  gate <= 7 most_x and lin <= 7 most_x + 2."""
    from rust_llm_inference_server_b200 import ops
    g = torch.Generator().manual_seed(seed)
    W, I, E = 48, 144, 2
    x = torch.randint(1, most_x + 1, (T, W), generator=g).double()
    x[:, 2] = torch.randint(0, 3, (T,), generator=g).double()
    up, down = torch.zeros(E, 2 * I, W, dtype=torch.float64), torch.zeros(E, W, I, dtype=torch.float64)
    for e in range(E):
        for i in range(I // 2):
            a, b = (int(v) for v in torch.randint(3, W, (2,), generator=g))
            c, d = (int(v) for v in torch.randint(1, 8, (2,), generator=g))
            up[e, 2 * i:2 * i + 2, a] = c
            up[e, I + 2 * i:I + 2 * i + 2, b] = d
            up[e, I + 2 * i, 2] = 1
        for f in range(W):
            i = int(torch.randint(0, I // 2, (1,), generator=g))
            down[e, f, 2 * i], down[e, f, 2 * i + 1] = 1, -1
    router = torch.zeros(E, W)
    router[0, 3], router[1, 4] = 1, 1
    want = torch.zeros(T, W, dtype=torch.float64)
    for t in range(T):
        e = 0 if x[t, 3] >= x[t, 4] else 1
        gate, lin = up[e, :I] @ x[t], up[e, I:] @ x[t]
        want[t] = down[e] @ (gate.clamp(min=0) * lin)
    if blocks:
        as_codes = lambda m: ops.BlockMatrix(m.float().cuda().to(torch.float8_e4m3fn), torch.ones(m.shape[0], -(-m.shape[1] // 128), -(-m.shape[2] // 128), device="cuda"))
    else:
        as_codes = lambda m: m.bfloat16().cuda()
    y = ops.moe_layer(x.bfloat16().cuda(), router.cuda(), as_codes(up), as_codes(down), 1, scoring="softmax_chosen", slope=float("inf"))
    return y.cpu(), want


# beside codes the gated results have up to 20 bits (889 * 891) of the 22 that two float16 hold; beside bfloat16 up to 16 (217 * 219), which two bfloat16 hold
@pytest.mark.parametrize("blocks,most_x", [(True, 127), (False, 31)])
@pytest.mark.parametrize("T", [1, 5, 8, 13, 16])
def test_gated_results_keep_their_last_digits(T, blocks, most_x):
    for seed in range(3):
        y, want = whole_layer(T, blocks, most_x, seed)
        assert torch.equal(y, want.bfloat16())
