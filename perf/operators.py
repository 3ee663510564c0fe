"""Products with weights in 8 bits, and a routed feed-forward of a few tokens as one call: what a change of their speed is measured on.

Four kinds of case.  "rows": a step's activations into e4m3 with a float32 scale for each block of 128 of a row.  "matrix": a weight into e4m3 with a float32
scale for each block of 128 x 128.  "linear": y = x @ w^T with both in that form (x quantised within the call, or, "given", by whoever made it, for several
products).  "layer": a whole mixture of experts for up to 16 tokens (router, choice, gated experts, the sum, a shared expert beside them), weights in bfloat16
or in blocks.

A block's scale is max(amax, 2^-100) / 448, and its codes are the e4m3 nearest to 448 x / max(amax, 2^-100): rounded once, since a quotient of two bfloat16
numbers often lies right between two e4m3.  Everything is made from the seed on the GPU: weights N(0, 0.02), activations as a norm leaves them, a few of
their channels twenty times as large."""

import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 128
FINITE = 448.0              # the largest e4m3
LEAST = 2.0 ** -100         # a block whose values are all smaller counts as this large
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # The step of eight users at the width of the benchmark's Llama 1B, before its attention.
        dict(name="rows_8", kind="rows", tokens=8, k=2048, dtype="bfloat16", wider=0),
        # A prompt's gated activations at the 8B sizes, which are the second half of wider rows.
        dict(name="rows_2048", kind="rows", tokens=2048, k=14336, dtype="bfloat16", wider=14336),
        # Weights at load time: a projection whose sizes fill no block, and the 1B sizes' gate|up matrix in the checkpoint's 32 bits.
        dict(name="matrix_odd", kind="matrix", rows=1000, k=1500, dtype="bfloat16"),
        dict(name="matrix_gate_up", kind="matrix", rows=16384, k=2048, dtype="float32"),
        # One user's token through the 1B sizes' output projection: the smallest product, all latency.
        dict(name="linear_1", kind="linear", tokens=1, n=2048, k=2048, dtype="bfloat16", out="bfloat16", given=False),
        # Eight users through its gate|up matrix, and 64 through the 8B sizes' down projection, in 32 bits for the residual stream.
        dict(name="linear_8", kind="linear", tokens=8, n=16384, k=2048, dtype="bfloat16", out="bfloat16", given=False),
        dict(name="linear_64", kind="linear", tokens=64, n=4096, k=14336, dtype="bfloat16", out="float32", given=False),
        # A portion of a prompt whose rows were quantised once for several products, sizes that fill no tile.
        dict(name="linear_509", kind="linear", tokens=509, n=6100, k=4000, dtype="bfloat16", out="bfloat16", given=True),
        # The headline prompt through the gate|up matrix.
        dict(name="linear_2048", kind="linear", tokens=2048, n=16384, k=2048, dtype="bfloat16", out="bfloat16", given=False),
        # The benchmark's routed layer: 4 of 32 experts beside a gated shared one; one user, and eight.
        dict(name="layer_1", kind="layer", tokens=1, width=2048, inner=1024, experts=32, top=4, scoring="sigmoid", normalize=False, shared=1024, blocks=False),
        dict(name="layer_8", kind="layer", tokens=8, width=2048, inner=1024, experts=32, top=4, scoring="sigmoid", normalize=False, shared=1024, blocks=False),
        # 16 users, 8 of 128 small experts by a normalised softmax, weights in blocks.
        dict(name="layer_16_blocks", kind="layer", tokens=16, width=2048, inner=768, experts=128, top=8, scoring="softmax", normalize=True, shared=0, blocks=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "matrix", "linear", "linear", "linear", "linear", "layer", "layer", "layer"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if kind == "rows":
        k = _log(rng, 64, 16384) if rng.random() < 0.5 else 128 * _log(rng, 1, 112)
        return dict(kind=kind, tokens=_log(rng, 1, 29_000_000 // k if k > 7200 else 4096), k=k, dtype=dtype, wider=rng.choice([0, 0, 1, 8, 512, k]))
    if kind == "matrix":
        k = _log(rng, 64, 16384) if rng.random() < 0.5 else 128 * _log(rng, 1, 112)
        return dict(kind=kind, rows=_log(rng, 16, min(16384, 33_000_000 // k)), k=k, dtype=dtype)
    if kind == "linear":
        k = _log(rng, 64, 16384) if rng.random() < 0.4 else 128 * _log(rng, 2, 112)
        n = _log(rng, 16, 30000) if rng.random() < 0.4 else 8 * _log(rng, 32, 2500)
        most = min(4096, 68_000_000_000 // (k * n))
        return dict(kind=kind, tokens=_log(rng, 1, rng.choice([16, 128, 4096]) if most > 4000 else most), n=n, k=k, dtype=dtype,
                    out=rng.choice(["bfloat16", "bfloat16", "float32"]), given=rng.random() < 0.3)
    width, top = rng.choice([1, 1, 2]) * 64 * _log(rng, 4, 32), rng.randint(1, 8)
    inner, experts = 32 * _log(rng, 4, 48), _log(rng, max(8, top), 128)
    while experts * inner * width > 220_000_000:
        experts, inner = max(8, top, experts // 2), max(128, inner - 128)
    return dict(kind=kind, tokens=_log(rng, 1, 16), width=width, inner=inner, experts=experts, top=top,
                scoring=rng.choice(["sigmoid", "softmax", "softmax_chosen"]), normalize=rng.random() < 0.4,
                shared=rng.choice([0, 0, inner, 2 * inner]), blocks=rng.random() < 0.5)


# ---- what a program has in hand -------------------------------------------------------------------------------------------------------


def _generator(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed((seed * 1000003 + sum((i + 1) * 7919 * (case.get(name, 0) + 1) for i, name in enumerate(("tokens", "k", "n", "rows", "width", "inner", "experts")))) % (1 << 62))
    return g


def _activations(g, tokens, k, dtype, wider=0):
    x = torch.randn((tokens, k + wider), generator=g, device=DEVICE)
    x *= torch.where(torch.rand((k + wider,), generator=g, device=DEVICE) < 0.01, 20.0, 1.0)
    return x.to(dtype)[:, wider:]


def _weight(g, shape, dtype=torch.bfloat16):
    return (0.02 * torch.randn(shape, generator=g, device=DEVICE)).to(dtype)


def _as_blocks(w):
    """A stored matrix (or a stack of them) in blocks: codes, whose rows start at multiples of 16 bytes, and scales, as a checkpoint brings them."""
    k = w.shape[-1]
    codes, scales = _codes(w, BLOCK)
    room = codes.new_zeros(codes.shape[:-1] + (k + -k % 16,))
    room[..., :k] = codes
    return room[..., :k], scales


def prepare(case, seed):
    g, kind = _generator(case, seed), case["kind"]
    if kind == "rows":
        return dict(kind=kind, x=_activations(g, case["tokens"], case["k"], TYPES[case["dtype"]], case["wider"]))
    if kind == "matrix":
        return dict(kind=kind, w=_weight(g, (case["rows"], case["k"]), TYPES[case["dtype"]]))
    if kind == "linear":
        x = _activations(g, case["tokens"], case["k"], TYPES[case["dtype"]])
        state = dict(kind=kind, x=x, w=_as_blocks(_weight(g, (case["n"], case["k"]))), out=TYPES[case["out"]], given=case["given"])
        if case["given"]:
            codes, scales = _as_blocks_of_rows(x)
            state["rows"] = (codes, scales)
        if own:
            from rust_llm_inference_server_b200 import ops
            state["weight"] = ops.BlockMatrix(*state["w"])
            if case["given"]:
                state["x"] = ops.BlockRows(*state["rows"])
        return state
    W, I, E, S = case["width"], case["inner"], case["experts"], case["shared"]
    state = dict(kind=kind, x=_activations(g, case["tokens"], W, torch.bfloat16), router=_weight(g, (E + (1 if S else 0), W), torch.float32),
                 correction=0.02 * torch.randn((E,), generator=g, device=DEVICE) if case["scoring"] == "sigmoid" else None, top=case["top"],
                 scoring=case["scoring"], normalize=case["normalize"], experts=E, blocks=case["blocks"])
    shapes = {"up": (E, 2 * I, W), "down": (E, W, I)}
    if S:
        shapes.update({"shared_up": (2 * S, W), "shared_down": (W, S)})
    for name, shape in shapes.items():
        w = _weight(g, shape)
        state[name] = _as_blocks(w) if case["blocks"] else w
    if own:
        from rust_llm_inference_server_b200 import ops
        state["weights"] = {n: ops.BlockMatrix(*state[n]) if case["blocks"] else state[n] for n in shapes}
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------


def _codes(x, rows):
    """Codes and scales of x [.., R, K] by blocks of `rows` x 128, in float32."""
    R, K = x.shape[-2:]
    padded = torch.nn.functional.pad(x.float(), (0, -K % BLOCK, 0, -R % rows))
    tiles = padded.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, rows))                  # [.., row block, row, k block, k]
    amax = tiles.abs().amax(dim=(-3, -1)).clamp(min=LEAST)                               # [.., row block, k block]
    codes = (tiles * FINITE / amax[..., :, None, :, None]).flatten(-2).flatten(-3, -2)[..., :R, :K]
    return codes.to(torch.float8_e4m3fn), amax / torch.full_like(amax, FINITE)           # (by a number, it would be a product with the number's reciprocal)


def _as_blocks_of_rows(x):
    """Codes whose rows start at multiples of 16 bytes, and scales [k block, token]."""
    T, K = x.shape
    codes, scales = _codes(x, 1)
    room = codes.new_zeros((T, K + -K % 16))
    room[:, :K] = codes
    return room[:, :K], scales.t().contiguous()


def _values(codes, scales, rows):
    """What codes and scales stand for."""
    R, K = codes.shape[-2:]
    return codes.float() * scales.repeat_interleave(rows, dim=-2)[..., :R, :].repeat_interleave(BLOCK, dim=-1)[..., :K]


def _matrix(w):
    return _values(*w, BLOCK) if isinstance(w, tuple) else w.float()


def _unit(x, w_gate_up, w_down):
    """A gated unit of every token, x [.., W] with matrices of its own: gate rows first, then the linear branch's."""
    gate, up = (w_gate_up @ x.unsqueeze(-1)).squeeze(-1).chunk(2, dim=-1)
    return (w_down @ (gate / (1.0 + torch.exp(-gate)) * up).unsqueeze(-1)).squeeze(-1)


def _chosen(w, idx):
    return _values(w[0][idx], w[1][idx], BLOCK) if isinstance(w, tuple) else w[idx].float()


def _layer(s):
    x, E = s["x"].float(), s["experts"]
    z = x @ s["router"].t()
    z, gate = z[:, :E], z[:, E:]
    score = z if s["scoring"] == "softmax_chosen" else 1.0 / (1.0 + torch.exp(-z)) if s["scoring"] == "sigmoid" else _softmax(z)
    choice = score if s["correction"] is None else score + s["correction"]
    idx = torch.sort(choice, dim=1, descending=True, stable=True)[1][:, :s["top"]]
    weight = score.gather(1, idx)
    if s["scoring"] == "softmax_chosen":
        weight = _softmax(weight)
    elif s["normalize"]:
        weight = weight / (weight.sum(1, keepdim=True) + 1e-20)
    y = _unit(x[:, None, :].expand(-1, s["top"], -1), _chosen(s["up"], idx), _chosen(s["down"], idx))
    out = (weight[:, :, None] * 2.5 * y).sum(1)
    if "shared_up" in s:
        out = out + 1.0 / (1.0 + torch.exp(-gate)) * _unit(x, _matrix(s["shared_up"]), _matrix(s["shared_down"]))
    return out.to(torch.bfloat16)


def _softmax(z):
    e = torch.exp(z - z.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def run(state):
    kind = state["kind"]
    if own:
        from rust_llm_inference_server_b200 import ops
        if kind == "rows":
            r = ops.quantize_rows(state["x"])
            return {"codes": r.values, "scales": r.scales}
        if kind == "matrix":
            m = ops.quantize_matrix(state["w"])
            return {"codes": m.values, "scales": m.scales}
        if kind == "linear":
            return ops.linear_blocks(state["x"], state["weight"], state["out"])
        w = state["weights"]
        return ops.moe_layer(state["x"], state["router"], w["up"], w["down"], state["top"], 2.5, correction=state["correction"], scoring=state["scoring"],
                             normalize=state["normalize"], shared=(w["shared_up"], w["shared_down"]) if "shared_up" in w else None, shared_gate="shared_up" in w)
    if kind == "rows":
        codes, scales = _codes(state["x"], 1)
        return {"codes": codes, "scales": scales.t().contiguous()}
    if kind == "matrix":
        codes, scales = _codes(state["w"], BLOCK)
        return {"codes": codes, "scales": scales}
    if kind == "linear":
        x = _values(*(state["rows"][0], state["rows"][1].t()) if state["given"] else _codes(state["x"], 1), 1)
        return (x @ _matrix(state["w"]).t()).to(state["out"])
    return _layer(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], 4 if case.get("dtype") == "float32" else 2
    blocks = lambda n: -(-n // BLOCK)
    if kind == "rows":
        return {"bytes": case["tokens"] * (case["k"] * (size + 1.0) + 4.0 * blocks(case["k"])), "flops": 0.0}
    if kind == "matrix":
        return {"bytes": case["rows"] * case["k"] * (size + 1.0) + 4.0 * blocks(case["rows"]) * blocks(case["k"]), "flops": 0.0}
    if kind == "linear":
        T, N, K = case["tokens"], case["n"], case["k"]
        rows = T * (K + 4.0 * blocks(K)) if case["given"] else 1.0 * T * K * size
        return {"bytes": rows + 1.0 * N * K + 4.0 * blocks(N) * blocks(K) + T * N * (4 if case["out"] == "float32" else 2), "flops": 2.0 * T * N * K}
    T, W, I, E, top, S = (case[n] for n in ("tokens", "width", "inner", "experts", "top", "shared"))
    used = E * (1.0 - (1.0 - top / E) ** T)              # experts that T tokens choose on average
    per = 1.0 + 4.0 / BLOCK ** 2 if case["blocks"] else 2.0
    return {"bytes": 3.0 * W * (used * I + S) * per + 4.0 * W * (E + (1 if S else 0)) + 4.0 * T * W, "flops": 2.0 * T * W * (3.0 * (top * I + S) + E)}


# ---- the same in 64 bits --------------------------------------------------------------------------------------------------------------


def _exact_scales(blocks):
    """amax of the last axis, at least 2^-100, and the scale as float32 holds it."""
    amax = blocks.abs().max(dim=-1).values.double()
    amax = torch.where(amax < LEAST, torch.full_like(amax, LEAST), amax)
    return amax, (amax / 448).float()


def _exact_codes(x, amax):
    """The e4m3 nearest to 448 x / amax: three bits behind the leading one, steps of 2^-9 below 2^-6, ties to the even one."""
    q = 448 * x.double() / amax
    mantissa = torch.frexp(q)[0]                         # in [1/2, 1): q / mantissa is a power of two, exactly
    step = torch.where(q == 0, 0.0, q / mantissa / 16).clamp(min=2.0 ** -9)
    return torch.round(q / step) * step


def _exact_rows(x):
    """Values in 64 bits and scales of rows by blocks of 128, a block of columns at a time."""
    parts, scales = [], []
    for piece in torch.split(x, BLOCK, dim=1):
        amax, s = _exact_scales(piece)
        parts.append(_exact_codes(piece, amax[:, None]))
        scales.append(s)
    return parts, scales


def _exact_matrix(w):
    parts, scales = [], []
    for band in torch.split(w, BLOCK, dim=0):
        row, row_scales = [], []
        for piece in torch.split(band, BLOCK, dim=1):
            amax, s = _exact_scales(piece.reshape(1, -1))
            row.append(_exact_codes(piece, amax[:, None]))
            row_scales.append(s)
        parts.append(torch.cat(row, 1))
        scales.append(torch.cat(row_scales))
    return torch.cat(parts, 0), torch.stack(scales)


def _stored(w):
    """A stored matrix in 64 bits."""
    if not isinstance(w, tuple):
        return w.double()
    codes, scales = w
    out = codes.double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            out[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scales[i, j].double()
    return out


def _of(w, e):
    return (w[0][e], w[1][e]) if isinstance(w, tuple) else w[e]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rows":
        parts, scales = _exact_rows(s["x"])
        return {"codes": torch.cat(parts, 1), "scales": torch.stack(scales).double()}
    if case["kind"] == "matrix":
        values, scales = _exact_matrix(s["w"])
        return {"codes": values, "scales": scales.double()}
    if case["kind"] == "linear":
        if case["given"]:
            x = torch.cat([c.double() * v.double()[:, None] for c, v in zip(torch.split(s["rows"][0], BLOCK, dim=1), s["rows"][1])], 1)
        else:
            x = torch.cat([c * v.double()[:, None] for c, v in zip(*_exact_rows(s["x"]))], 1)
        w = s["w"][0].double()
        for j, column in enumerate(s["w"][1].double().t()):
            w[:, j * BLOCK:(j + 1) * BLOCK] *= column.repeat_interleave(BLOCK)[:w.shape[0], None]
        return torch.einsum("tk,nk->tn", x, w)
    x, E, top = s["x"].double(), s["experts"], s["top"]
    z = torch.einsum("tw,ew->te", x, s["router"].double())
    out = torch.zeros_like(x)
    for t in range(x.shape[0]):
        score = {"sigmoid": torch.sigmoid, "softmax": lambda v: torch.softmax(v, 0), "softmax_chosen": lambda v: v}[case["scoring"]](z[t, :E])
        rank = score + s["correction"].double() if s["correction"] is not None else score
        order = sorted(range(E), key=lambda e, r=rank.tolist(): (-r[e], e))[:top]
        weight = score[order]
        if case["scoring"] == "softmax_chosen":
            weight = torch.softmax(weight, 0)
        elif case["normalize"]:
            weight = weight / (weight.sum() + 1e-20)
        todo = [(_of(s["up"], e), _of(s["down"], e), 2.5 * c) for e, c in zip(order, weight)]
        if case["shared"]:
            todo.append((s["shared_up"], s["shared_down"], torch.sigmoid(z[t, E])))
        for up, down, c in todo:
            both = _stored(up) @ x[t]
            half = both.shape[0] // 2
            out[t] += c * (_stored(down) @ (both[:half] * torch.sigmoid(both[:half]) * both[half:]))
    return out
