"""A whole mixture of experts for a few tokens against the formulas in 64 bits, one token and one choice at a time."""

import math

import pytest
import torch

from tests.blocks_util import B, values_of

pytestmark = pytest.mark.gpu


def make(T, W, I, E, S=0, gate=False, identity=0, blocks=False, seed=0, scale=0.05):
    from rust_llm_inference_server_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T * 7 + W + I + E + seed)
    r = lambda *s: scale * torch.randn(*s, device="cuda", generator=g)
    m = dict(x=(20 * r(T, W)).bfloat16(), router=r(E + identity + (1 if gate else 0), W))
    shapes = {"up": (E, 2 * I, W), "down": (E, W, I)}
    if S:
        shapes.update(shared_up=(2 * S, W), shared_down=(W, S))
    for n, s in shapes.items():
        w = r(*s).bfloat16()
        m[n] = ops.quantize_matrix(w) if blocks else w
    return m


def call(m, top, scale=1.0, **more):
    from rust_llm_inference_server_b200 import ops
    shared = (m["shared_up"], m["shared_down"]) if "shared_up" in m else None
    return ops.moe_layer(m["x"], m["router"], m["up"], m["down"], top, scale, shared=shared, **more)


def plain(m, top, scale=1.0, correction=None, router_bias=None, scoring="sigmoid", groups=None, normalize=False, n_identity=0, shared_gate=False, slope=1.0, limit=None,
          up_shift=0.0, interleave=0, shared_interleave=0):
    """The layer in 64 bits, and for every result the sum of the sizes of what is added."""
    stored = {n: values_of(w.values.cpu(), w.scales.cpu(), B) if not isinstance(w, torch.Tensor) else w.double().cpu() for n, w in m.items() if n not in ("x", "router")}
    x, router = m["x"].double().cpu(), m["router"].double().cpu()
    E = stored["up"].shape[0]
    n = E + n_identity
    out, size, chosen = torch.zeros_like(x), torch.zeros_like(x), []

    def unit(up, down, v, il):
        I = up.shape[0] // 2
        rows = torch.arange(I)
        gr = rows // il * 2 * il + rows % il if il else rows
        gate, lin = up[gr] @ v, up[gr + (il or I)] @ v
        if limit is not None:
            gate, lin = gate.clamp(max=limit), lin.clamp(-limit, limit)
        h = (gate.clamp(min=0) if math.isinf(slope) else gate * torch.sigmoid(slope * gate)) * (lin + up_shift)
        return down @ h, down.abs() @ h.abs()

    for t in range(x.shape[0]):
        z = router @ x[t]
        if router_bias is not None:
            z[:n] += router_bias.double().cpu()
        s = torch.sigmoid(z[:n]) if scoring == "sigmoid" else torch.softmax(z[:n], 0) if scoring == "softmax" else z[:n]
        c = s + correction.double().cpu() if correction is not None else s.clone()
        if groups is not None:
            count, keep = groups
            best = c.view(count, -1).max(1).values.tolist()
            kept = sorted(range(count), key=lambda i: (-best[i], i))[:keep]
            c = torch.tensor([v if i // (n // count) in kept else -math.inf for i, v in enumerate(c.tolist())], dtype=torch.float64)
        order = sorted(range(n), key=lambda i, c=c.tolist(): (-c[i], i))[:top]
        w = s[order]
        if scoring == "softmax_chosen":
            w = torch.softmax(w, 0)
        elif normalize:
            w = w / (w.sum() + 1e-20)
        for e, v in zip(order, (w * scale).tolist()):
            y, a = unit(stored["up"][e], stored["down"][e], x[t], interleave) if e < E else (x[t], x[t].abs())
            out[t] += v * y
            size[t] += abs(v) * a
        if "shared_up" in stored:
            y, a = unit(stored["shared_up"], stored["shared_down"], x[t], shared_interleave)
            v = float(torch.sigmoid(z[n])) if shared_gate else 1.0
            out[t] += v * y
            size[t] += v * a
        chosen.append(order)
    return out, size, chosen


def close(y, m, want, size, top):
    """Where the sums of a unit's first product are off by r of themselves, its gated result is off by about 3 r of its size at this data's sums (silu and the
    product), and pairs of bfloat16 by 2^-17; the second sum by its own roundings.  Beside codes h is float16: every value is off by up to 2^-11 of it, their sum with
    the second matrix by 2^-11 of the sum of sizes.  Sums of K terms in float32, in the order of tensor-core steps: half a unit
    for each of K / 16 + 16 additions, of the sum of sizes, which is up to about sqrt(K) of the sum."""
    K = max(m["x"].shape[1], 256)
    r = (K / 16 + 24) * 2.0 ** -23
    bound = (3 * r * math.sqrt(K) / 4 + (2.0 ** -16 if isinstance(m["up"], torch.Tensor) else 2.0 ** -11) + r) * size
    bound = bound + 2.0 ** -8 * (want.abs() + bound) + 1e-30
    y = y.double().cpu()
    assert bool(((y - want).abs() <= bound).all()), float(((y - want).abs() / bound).max())


# one token, the edge of the first eight columns and of the tokens; widths that end inside a chunk and a warp's turn; experts fewer than a cluster's CTAs and more than
# eight for each; one feature group and a few
@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("T,W,I,E,top,S", [(1, 16, 16, 1, 1, 0), (1, 2048, 128, 6, 2, 64), (3, 2064, 48, 5, 2, 0), (8, 1936, 16, 8, 4, 16), (1, 256, 128, 8, 2, 0), (3, 272, 48, 5, 5, 32), (8, 512, 256, 32, 4, 256), (9, 128, 64, 40, 3, 0),
                                           (16, 384, 96, 70, 8, 160), (16, 2304, 32, 3, 2, 16), (7, 4112, 16, 9, 1, 0), (2, 1024, 144, 512, 16, 0)])
def test_layers(blocks, T, W, I, E, top, S):
    m = make(T, W, I, E, S, gate=S > 0, blocks=blocks)
    want, size, _ = plain(m, top, 2.5, shared_gate=S > 0)
    y = call(m, top, 2.5, shared_gate=S > 0)
    assert y.shape == (T, W) and y.dtype == torch.bfloat16
    close(y, m, want, size, top)
    assert torch.equal(call(m, top, 2.5, shared_gate=S > 0), y)             # no order that timing decides


# more of the experts' results than shared memory holds at a time: one go of output features, and two; and experts that fill it alone
@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("T,W,I,E,top,S", [(16, 64, 4096, 16, 8, 0), (16, 2304, 2048, 4, 4, 1040), (9, 48, 16384, 2, 2, 0), (16, 32, 4112, 1, 1, 8192)])
def test_layers_in_several_goes(blocks, T, W, I, E, top, S):
    m = make(T, W, I, E, S, blocks=blocks, scale=0.02)
    want, size, _ = plain(m, top)
    close(call(m, top), dict(m, x=torch.empty(1, max(W, I, S))), want, size, top)


@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("how", [
    dict(scoring="softmax"), dict(scoring="softmax", normalize=True, correction=True), dict(scoring="softmax_chosen", router_bias=True), dict(normalize=True, router_bias=True),
    dict(groups=(4, 2), correction=True), dict(n_identity=8, scoring="softmax"), dict(n_identity=4, groups=(2, 1), shared_gate=True), dict(slope=float("inf")),
    dict(slope=1.7, limit=0.3, up_shift=1.0), dict(interleave=4), dict(interleave=8, shared_interleave=4, shared_gate=True), dict(scoring="softmax", shared_gate=True)])
def test_ways_to_route_and_to_gate(blocks, how):
    how = dict(how)
    n = 12 + how.get("n_identity", 0)
    g = torch.Generator(device="cuda").manual_seed(n)
    for name in ("correction", "router_bias"):
        if how.get(name):
            how[name] = torch.randn(n, device="cuda", generator=g)
    for T in (1, 5, 13):
        m = make(T, 256, 64, 12, 64 if T != 5 or how.get("shared_gate") or how.get("shared_interleave") else 0, how.get("shared_gate", False), how.get("n_identity", 0), blocks, T)
        want, size, _ = plain(m, 3, 1.5, **how)
        close(call(m, 3, 1.5, **how), m, want, size, 3)


def test_ties_go_to_the_lower_index_and_nan_is_not_chosen():
    m = make(4, 64, 16, 6)
    m["router"][:] = 0.0                    # all scores 1/2
    want, size, chosen = plain(m, 3)
    assert chosen == [[0, 1, 2]] * 4
    close(call(m, 3), m, want, size, 3)
    correction = torch.tensor([0.0, -0.0, float("nan"), 0.0, float("-inf"), 0.0], device="cuda")
    want, size, _ = plain(m, 3, correction=torch.tensor([0.0, 0.0, -1.0, 0.0, -1.0, 0.0]))
    close(call(m, 3, correction=correction), m, want, size, 3)
    # nothing compares: outputs in order, none twice
    nan = torch.full((6,), float("nan"), device="cuda")
    want, size, _ = plain(m, 3)
    close(call(m, 3, correction=nan), m, want, size, 3)
    want, size, _ = plain(m, 6)
    close(call(m, 6, correction=torch.full((6,), float("-inf"), device="cuda")), m, want, size, 6)


@pytest.mark.parametrize("blocks", [False, True])
def test_a_token_that_is_no_number_leaves_the_others(blocks):
    m = make(9, 128, 64, 8, 32, blocks=blocks)
    clean = call(m, 2)
    m["x"][4, 17] = float("nan")
    y = call(m, 2)
    assert bool(y[4].isnan().all()) and torch.equal(y[[0, 1, 2, 3, 5, 6, 7, 8]], clean[[0, 1, 2, 3, 5, 6, 7, 8]])
    m["x"][4, 17] = float("inf")
    assert torch.equal(call(m, 2)[[0, 8]], clean[[0, 8]])


@pytest.mark.parametrize("T", [5, 13])
@pytest.mark.parametrize("blocks", [False, True])
def test_weights_that_are_no_numbers_reach_only_who_chose_them(blocks, T):
    from rust_llm_inference_server_b200 import ops
    m = make(T, 144, 80, 6, 32, blocks=blocks)
    clean, (_, _, chosen) = call(m, 2), plain(m, 2)
    e = next(e for e in range(6) if 0 < sum(e in c for c in chosen) < T)
    who = torch.tensor([e in c for c in chosen], device="cuda")
    for name, at in (("up", (e, 70, 143)), ("down", (e, 33, 79)), ("down", (e, 16, 0))):
        bad = dict(m)
        if blocks:
            codes = m[name].values.clone().view(torch.uint8)
            codes[at] = 127
            bad[name] = ops.BlockMatrix(codes.view(torch.float8_e4m3fn), m[name].scales)
        else:
            bad[name] = m[name].clone()
            bad[name][at] = float("inf") if at[1] == 16 else float("nan")
        y = call(bad, 2)
        assert torch.equal(y[~who], clean[~who])
        touched = y[who] if name == "up" else y[who][:, at[1]]
        assert not bool(touched.isfinite().any())


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e12])
@pytest.mark.parametrize("blocks", [False, True])
def test_activations_of_any_size(blocks, size):
    """Rows far from one, each of its own size, and values far below a row's largest."""
    m = make(6, 256, 64, 8, 32, blocks=blocks)
    m["router"] *= 0.0              # (so that their size decides nothing about the choice)
    m["x"] = (m["x"].float() * size * 10.0 ** torch.arange(-2, 4, device="cuda")[:, None] * (4.0 ** -torch.arange(256, device="cuda").remainder(12))).bfloat16()
    want, size_of, _ = plain(m, 3)
    close(call(m, 3), m, want, size_of, 3)


@pytest.mark.parametrize("blocks", [False, True])
def test_all_tokens_at_one_expert_and_rows_inside_wider_ones(blocks):
    m = make(16, 256, 64, 8, 0, blocks=blocks)
    correction = torch.zeros(8, device="cuda")
    correction[5] = 10.0
    want, size, chosen = plain(m, 1, correction=correction)
    assert chosen == [[5]] * 16
    y = call(m, 1, correction=correction)
    close(y, m, want, size, 1)
    wide = torch.full((16, 280), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 8:264] = m["x"]
    m["x"] = wide[:, 8:264]
    out = torch.full((18, 256), 7.0, device="cuda", dtype=torch.bfloat16)
    from rust_llm_inference_server_b200 import ops
    got = ops.moe_layer(m["x"], m["router"], m["up"], m["down"], 1, correction=correction, out=out[1:17])
    assert torch.equal(got, y) and got.data_ptr() == out[1:].data_ptr() and bool((out[0] == 7).all()) and bool((out[17] == 7).all())


def test_the_layer_is_what_its_parts_are():
    """The layer beside moe_route, moe_up, moe_down and moe_combine, whose activations between are rounded to bfloat16 (2^-8 of a half each)."""
    from rust_llm_inference_server_b200 import ops

    class Step:
        def buffer(self, name, shape, dtype):
            return torch.empty(shape, dtype=dtype, device="cuda")

    m = make(8, 512, 256, 32)
    plan = ops.moe_route(m["x"], m["router"], None, 32, 4, 2.5, False, Step())
    act = ops.moe_up(m["x"], m["up"], plan, 1.0, float("inf"), 0.0, Step())
    parts = ops.moe_combine(ops.moe_down(act, m["down"], plan, Step()), plan, None, torch.empty_like(m["x"]))
    want, size, _ = plain(m, 4, 2.5)
    assert bool(((call(m, 4, 2.5).double().cpu() - parts.double().cpu()).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -7 * size).all())


def test_codes_and_scales_from_a_checkpoint():
    """Every e4m3 there is, NaN left to its own row, and scales of either sign."""
    from rust_llm_inference_server_b200 import ops
    m = make(3, 256, 32, 4, blocks=True)
    every = torch.arange(256, device="cuda").to(torch.uint8)
    every[127], every[255] = 0, 0
    up = m["up"].values.clone().view(torch.uint8)
    up[:, 5, :] = every
    up[:, 37, :] = every.flip(0)
    m["up"] = ops.BlockMatrix(up.view(torch.float8_e4m3fn), m["up"].scales * torch.tensor([[1.0, -0.5]], device="cuda"))
    want, size, _ = plain(m, 4)
    y = call(m, 4)
    close(y, m, want, size, 4)
    down = m["down"].values.clone().view(torch.uint8)
    down[2, 9, 17] = 127                            # NaN: its feature, for every token that chose the expert (all)
    m["down"] = ops.BlockMatrix(down.view(torch.float8_e4m3fn), m["down"].scales)
    z = call(m, 4)
    rest = torch.arange(256, device="cuda") != 9
    assert bool(z[:, 9].isnan().all()) and torch.equal(z[:, rest], y[:, rest])


@pytest.mark.parametrize("blocks", [False, True])
def test_calls_at_once_and_from_a_graph(blocks):
    """Two streams, and two graphs whose replays lie side by side: every call has a workspace of its own."""
    ms = [make(4, 256, 64, 16, 64, True, blocks=blocks, seed=s) for s in (1, 2)]
    want = [call(m, 4, shared_gate=True) for m in ms]
    streams = [torch.cuda.Stream() for _ in ms]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (m, s) in enumerate(zip(ms, streams)):
            with torch.cuda.stream(s):
                got[i].append(call(m, 4, shared_gate=True))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for g, w in zip(got, want) for y in g)
    graphs, outs = [], []
    for m in ms:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(m, 4, shared_gate=True))
        graphs.append(g)
    x0 = ms[0]["x"].clone()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for y, w in zip(outs, want))
    ms[0]["x"].copy_(x0.flip(0))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0].flip(0))


def test_refused_calls():
    from rust_llm_inference_server_b200 import ops
    from rust_llm_inference_server_b200.ops import KernelError
    m = make(2, 128, 32, 4, 32)
    blocks = make(2, 128, 32, 4, 32, blocks=True)
    assert ops.moe_layer(m["x"][:0], m["router"], m["up"], m["down"], 2).shape == (0, 128)
    f = lambda **c: ops.moe_layer(*[c.get(n, m[n]) for n in ("x", "router", "up", "down")], c.get("top", 2), **{n: v for n, v in c.items() if n not in ("x", "router", "up", "down", "top")})
    f()
    for c in (dict(x=make(17, 128, 32, 4)["x"]), dict(x=m["x"].float()), dict(x=m["x"].cpu()), dict(x=m["x"][:, :120]), dict(router=m["router"].bfloat16()), dict(router=m["router"][:3]),
              dict(up=blocks["up"]), dict(down=blocks["down"]), dict(up=m["up"][:, :62]), dict(down=m["down"][:3]), dict(up=m["up"].float()), dict(top=0), dict(top=5), dict(top=17),
              dict(scoring="relu"), dict(groups=(3, 1)), dict(groups=(4, 1)), dict(groups=(2, 3)), dict(shared_gate=True), dict(shared=(m["shared_up"],  m["down"][0][:, :16])),
              dict(shared=(blocks["shared_up"], blocks["shared_down"])), dict(correction=torch.zeros(3, device="cuda")), dict(router_bias=torch.zeros(4)), dict(interleave=5),
              dict(interleave=-1), dict(out=torch.empty(2, 128, device="cuda")), dict(n_identity=1), dict(x=torch.zeros(2, 129, device="cuda", dtype=torch.bfloat16)[:, 1:])):
        with pytest.raises(KernelError):
            f(**c)
    with pytest.raises(KernelError):
        ops.moe_layer(blocks["x"], blocks["router"], blocks["up"], blocks["down"], 2, interleave=2)
