"""The ops in blocks as a step uses them: one after the other, in a captured graph, on several streams at once, on empty and on very long tensors."""

import pytest
import torch

from tests.test_blocks_gpu import close as product_close
from tests.test_moe_layer_gpu import close as layer_close, plain as plain_layer

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(sum((i + 1) * s for i, s in enumerate(shape)) + seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


def weights(W=256, I=128, E=8, S=64):
    from rust_llm_inference_server_b200 import ops
    q = lambda *s: ops.quantize_matrix(rand(*s, scale=s[-1] ** -0.5))
    return dict(qkv=q(3 * W, W), proj=q(W, W), router=rand(E, W, scale=0.1, dtype=torch.float32), up=q(E, 2 * I, W), down=q(E, W, I), shared=(q(2 * S, W), q(W, S)))


def step(x, w):
    """A layer's products: two of the same rows in blocks, a third of plain ones, and the experts.  What each of them gave."""
    from rust_llm_inference_server_b200 import ops
    rows = ops.quantize_rows(x)
    a, b = ops.linear_blocks(rows, w["qkv"], torch.float32, early=True), ops.linear_blocks(rows, w["proj"], early=True)
    W = x.shape[1]
    mixed = (a[:, :W] + a[:, W:2 * W] * torch.sigmoid(a[:, 2 * W:])).bfloat16()
    c = ops.linear_blocks(mixed, w["proj"])
    v = b + c
    return a, b, mixed, c, v, ops.moe_layer(v, w["router"], w["up"], w["down"], 2, shared=w["shared"])


@pytest.mark.parametrize("T", [1, 5, 16])
def test_a_step_of_them(T):
    """Each op against 64 bits on what the one before it gave, so that a rounding of one cannot pass for an error of the next."""
    from rust_llm_inference_server_b200 import ops
    w, x = weights(), rand(T, 256)
    a, b, mixed, c, v, y = step(x, w)
    rows = ops.quantize_rows(x)
    product_close(a, rows, w["qkv"], torch.float32)
    product_close(b, rows, w["proj"], torch.bfloat16)
    product_close(c, ops.quantize_rows(mixed), w["proj"], torch.bfloat16)
    layer = dict(x=v, router=w["router"], up=w["up"], down=w["down"], shared_up=w["shared"][0], shared_down=w["shared"][1])
    want, size, _ = plain_layer(layer, 2)
    layer_close(y, layer, want, size, 2)
    ops.check_device_errors()


def test_steps_from_graphs_and_on_two_streams():
    """Two captured steps of the same weights replayed side by side, beside a step that is not captured: scratch and workspaces are a call's own."""
    w = weights()
    xs = [rand(T, 256, seed=T) for T in (3, 16)]
    want = [step(x, w)[-1] for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x, w)[-1])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        assert torch.equal(step(xs[0], w)[-1], want[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    xs[0].copy_(xs[1][:3])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], step(xs[0], w)[-1]) and not torch.equal(outs[0], want[0])


@pytest.mark.parametrize("M", [1, 40, 100, 200, 600])
def test_products_on_two_streams_and_from_graphs(M):
    from rust_llm_inference_server_b200 import ops
    ws = [ops.quantize_matrix(rand(n, 1700, scale=0.03)) for n in (700, 1000)]
    x = rand(M, 1700)
    want = [ops.linear_blocks(x, w, torch.float32) for w in ws]
    streams = [torch.cuda.Stream() for _ in ws]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (w, s) in enumerate(zip(ws, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.linear_blocks(x, w, torch.float32))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    assert all(torch.equal(y, v) for g, v in zip(got, want) for y in g)
    with torch.cuda.graph(graph):
        rows = ops.quantize_rows(x)
        captured = [ops.linear_blocks(rows, w, torch.float32, early=True) for w in ws] + [ops.linear_blocks(x, ws[0], torch.float32)]
    for v in (x.clone(), x.flip(0)):
        x.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, ops.linear_blocks(x, w, torch.float32)) for a, w in zip(captured, ws + ws[:1]))
    ops.check_device_errors()


def test_a_weight_written_right_before_its_product():
    """Rows of another step's result, a weight that the kernel before has just made: nothing is read before it is written."""
    from rust_llm_inference_server_b200 import ops
    for M in (8, 300):
        x, w = rand(M, 1024), rand(2048, 1024, scale=0.03)
        m = ops.quantize_matrix(w)
        want = ops.linear_blocks(x, m)
        torch.cuda.synchronize()
        for i in range(20):
            made = ops.quantize_matrix(w * 2.0 ** i)
            assert torch.equal(ops.linear_blocks(x, made), (want.float() * 2.0 ** i).bfloat16())
            made = ops.quantize_matrix(w)
            assert torch.equal(ops.linear_blocks(ops.quantize_rows(x), made), want)


@pytest.mark.parametrize("blocks", [False, True])
def test_experts_written_right_before_their_layer(blocks):
    from rust_llm_inference_server_b200 import ops
    T, W, I, E, S = 6, 1024, 256, 8, 512
    x, router = rand(T, W), rand(E, W, scale=0.1, dtype=torch.float32)
    plain = [rand(*s, scale=s[-1] ** -0.5) for s in ((E, 2 * I, W), (E, W, I), (2 * S, W), (W, S))]
    make = lambda: [ops.quantize_matrix(w) if blocks else w.clone() for w in plain]
    call = lambda up, down, a, b: ops.moe_layer(x, router, up, down, 2, shared=(a, b))
    want = call(*make())
    torch.cuda.synchronize()
    for _ in range(20):
        assert torch.equal(call(*make()), want)
        made = make()[::-1]                                 # the last written is the first used
        assert torch.equal(call(*made[::-1]), want)


def test_tensors_without_rows():
    from rust_llm_inference_server_b200 import ops
    none = ops.quantize_matrix(rand(0, 96))
    assert none.shape == (0, 96) and none.scales.shape == (0, 1) and ops.linear_blocks(rand(3, 96), none).shape == (3, 0)
    assert ops.quantize_matrix(rand(0, 8, 96)).shape == (0, 8, 96)
    rows = ops.quantize_rows(rand(0, 96))
    assert ops.linear_blocks(rows, ops.quantize_matrix(rand(5, 96))).shape == (0, 5)


def test_rows_whose_offsets_pass_32_bits():
    """2^32 and more codes: rows, a stack of matrices, and a product with a result of as many values."""
    from rust_llm_inference_server_b200 import ops
    T, K = 262_160, 16_400
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    ends = rand(40, K)
    x[:20], x[-20:] = ends[:20], ends[20:]
    r, few = ops.quantize_rows(x), ops.quantize_rows(ends)
    pick = lambda v: torch.cat([v[:20], v[-20:]])
    assert torch.equal(pick(r.values).view(torch.uint8), few.values.view(torch.uint8)) and torch.equal(pick(r.scales.t()), few.scales.t())
    m = ops.quantize_matrix(x.view(40, T // 40, K))
    last = ops.quantize_matrix(x[-(T // 40):])
    assert torch.equal(m.values[39].view(torch.uint8), last.values.view(torch.uint8)) and torch.equal(m.scales[39], last.scales)
    del m, last, x
    w = ops.quantize_matrix(rand(24, K))
    y = ops.linear_blocks(r, w)
    product_close(pick(y), few, w, torch.bfloat16)
    assert not bool(y[20:-20].any())
    del r, y
    thin = ops.quantize_rows(rand(262_160, 16))
    wide = ops.quantize_matrix(rand(16_401, 16))            # a row of results starts anywhere
    z = ops.linear_blocks(thin, wide)
    some = ops.BlockRows(thin.values[-300:], thin.scales[:, -300:].contiguous())
    assert torch.equal(z[-300:], ops.linear_blocks(some, wide))
    ops.check_device_errors()
