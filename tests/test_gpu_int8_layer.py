"""The 8-bit layer as a module: casts and moves, hooks, shared layers, and the model it was made from."""
import pytest
import torch

import kan_b200

pytestmark = pytest.mark.gpu


def a_layer(n_in=40, n_out=24, degree=3, seed=0):
    torch.manual_seed(seed)
    return kan_b200.ChebyKANLayer(n_in, n_out, degree).cuda()


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.float16),
                                  lambda m: m.to("cuda:0", torch.bfloat16), lambda m: m.type(torch.float16), lambda m: m.half().float()])
def test_casts_leave_the_packed_values(cast):
    layer = kan_b200.quantize_int8(a_layer())
    x = torch.randn(9, 40, device="cuda")
    with torch.no_grad():
        want = layer(x), layer(x.bfloat16())
        state = {k: v.clone() for k, v in layer.state_dict().items()}
        served = cast(layer)
        assert served is layer
        assert all(v.dtype == state[k].dtype and torch.equal(v, state[k]) for k, v in served.state_dict().items())
        assert torch.equal(served(x), want[0]) and torch.equal(served(x.bfloat16()), want[1])


def test_a_served_layer_moves_to_the_host_and_back():
    layer = kan_b200.quantize_int8(a_layer())
    x = torch.randn(9, 40, device="cuda")
    want = layer(x)
    layer.cpu()
    assert not any(b.is_cuda for b in layer.buffers())
    with pytest.raises(RuntimeError, match="CUDA"):
        layer(x)
    layer.half().cuda()
    assert torch.equal(layer(x), want)
