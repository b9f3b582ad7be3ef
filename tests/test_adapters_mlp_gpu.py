"""Gate and up with an adapter in a decode step: 32-bit sums up to the activation."""

import pytest
import torch

from reflex_b200 import InvalidInput, ops
from reflex_b200.config.spec import FeedForwardSpec
from reflex_b200.parts import FEED_FORWARDS

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 9, 64])
def test_what_an_adapter_leaves_of_the_shared_product(rows, dtype):
    """The gate's product is 1 + 2^-9 and the adapter's -1: what is left, 2^-9, is lost where the product is rounded to
    bfloat16.  The up's is 1, the down projection sums what is the same I times."""
    H, I = 64, 128
    spec = FeedForwardSpec("swiglu", hidden_size=H, intermediate_size=I)
    mlp = FEED_FORWARDS.get("swiglu")(spec, dtype, DEV)
    gate, up, down = torch.zeros(I, H), torch.zeros(I, H), torch.ones(H, I)
    gate[:, 0], gate[:, 1], up[:, 0] = 1.0, 1.0, 1.0
    mlp.bind({"gate_proj": gate.to(dtype), "up_proj": up.to(dtype), "down_proj": down.to(dtype)})
    a = torch.zeros(4, H)
    a[0, 0] = -1.0
    mlp.adapters = mlp.adapter_banks({"gate_proj": [(a, torch.eye(4)[:1].expand(I, 4).contiguous())]}, [1.0])
    x = torch.zeros(rows, H, device=DEV, dtype=dtype)
    x[:, 0], x[:, 1] = 1.0, 2.0 ** -9
    ids = torch.zeros(rows, dtype=torch.int32, device=DEV)
    with ops.use_adapters(ops.adapter_rows(ids, 1)):
        got = mlp.forward(x)
    g = torch.tensor(2.0 ** -9, dtype=torch.float64)
    want = float(I * torch.nn.functional.silu(g))
    # the activation is rounded once; its sum of 128 equal terms is exact but for a step of each
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    assert bool(((got.double() - want).abs() <= want * (half + (I + 8) * 2.0 ** -23)).all()), float(got.flatten()[0])


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("alternating", [False, True])
@pytest.mark.parametrize("R,I", [(1, 1), (5, 37), (64, 1024)])
def test_activations_of_32_bit_sums_in_bfloat16(R, I, alternating, activation):
    g = torch.Generator().manual_seed(R + I)
    gu = (torch.randn(R, 2 * I, generator=g) * 3).to(DEV)
    got = ops.swiglu(gu, alternating=alternating, activation=activation, out_dtype=torch.bfloat16)
    gate, up = (gu[:, 0::2], gu[:, 1::2]) if alternating else (gu[:, :I], gu[:, I:])
    gate = gate.double()
    act = torch.nn.functional.silu(gate) if activation == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
    want = act * up.double()
    assert got.dtype == torch.bfloat16
    # one rounding to bfloat16; of the activation's own 32-bit steps (an exponential, a quotient or tanh) 2^-11 is
    # far above any, gelu's tail cancels to steps of its argument
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -8 * (1 + 2.0 ** -3) + up.double().abs() * gate.abs() * 2.0 ** -20).all())


def test_types_that_do_not_go_together():
    gu = torch.zeros(2, 8, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(InvalidInput, match="does not go"):
        ops.swiglu(gu, out_dtype=torch.float32)
    with pytest.raises(InvalidInput, match="does not go"):
        ops.swiglu(gu.float(), out_dtype=torch.float16)
