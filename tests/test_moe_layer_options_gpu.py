"""The routed layer in the form in which the framework's own layer holds its experts and gates them: branches interleaved by 4, a slope, a limit and a shift together."""

import pytest
import torch

from tests.test_moe_layer_gpu import call, close, make, plain

pytestmark = pytest.mark.gpu

HOW = dict(interleave=4, slope=1.702, limit=0.3, up_shift=1.0)


class Step:
    def buffer(self, name, shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("T", [1, 8, 15])
@pytest.mark.parametrize("shared", [0, 96])
def test_the_form_of_the_framework_s_layer(T, blocks, shared):
    m = make(T, 384, 160, 12, shared, gate=shared > 0, blocks=blocks)
    how = dict(HOW, normalize=True, shared_gate=shared > 0, shared_interleave=4 if shared else 0)
    want, size, _ = plain(m, 4, 1.5, **how)
    # (what the limit cuts and the shift adds to is no sum of products: sizes count 1 for it, times the second matrix)
    down = m["down"] if not blocks else m["down"].values.float() * m["down"].scales.repeat_interleave(128, 1)[:, :384].repeat_interleave(128, 2)[:, :, :160]
    size = size + 1.5 * down.abs().double().sum(2).amax(0).cpu()
    close(call(m, 4, 1.5, **how), m, want, size, 4)


@pytest.mark.parametrize("T", [1, 8, 16])
def test_the_form_of_the_framework_s_layer_beside_its_parts(T):
    """Whose activations between are rounded to bfloat16 (2^-8 of each at most)."""
    from rust_llm_inference_server_b200 import ops
    m = make(T, 512, 256, 32)
    plan = ops.moe_route(m["x"], m["router"], None, 32, 4, 2.5, False, Step())
    act = ops.moe_up(m["x"], m["up"], plan, HOW["slope"], HOW["limit"], HOW["up_shift"], Step(), 4)
    parts = ops.moe_combine(ops.moe_down(act, m["down"], plan, Step()), plan, None, torch.empty_like(m["x"]))
    want, size, _ = plain(m, 4, 2.5, **HOW)
    assert bool(((call(m, 4, 2.5, **HOW).double().cpu() - parts.double().cpu()).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -7 * size).all())


# groups of rows that lie across the ends of blocks of 128, and that end inside the eight rows of a load
@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("I,S,il,shared_il", [(240, 48, 12, 12), (240, 80, 20, 4), (144, 0, 36, 0), (240, 240, 60, 120)])
def test_other_interleavings(blocks, I, S, il, shared_il):
    for T in (3, 12):
        m = make(T, 144, I, 5, S, blocks=blocks)
        want, size, _ = plain(m, 2, interleave=il, shared_interleave=shared_il)
        close(call(m, 2, interleave=il, shared_interleave=shared_il), m, want, size, 2)
