"""The 8-bit layer as a module: casts and moves, hooks, shared layers, and the model it was made from."""
import warnings

import pytest
import torch
import torch.nn.utils.parametrize
import torch.nn.utils.prune

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


class Scaled(torch.nn.Sequential):
    def __init__(self, *layers):
        super().__init__(*layers)
        self.register_buffer("factor", torch.tensor(2.0))

    def forward(self, x):
        return super().forward(x) * self.factor


def test_what_is_registered_with_the_served_model_stays_off_the_original():
    model = Scaled(a_layer(), Scaled(torch.nn.LayerNorm(24), a_layer(24, 8))).cuda()
    served = kan_b200.quantize_int8(model)
    seen = []
    for m in (served, served[1]):
        m.register_forward_hook(lambda *a: seen.append(1))
        m.register_forward_pre_hook(lambda *a: seen.append(1))
        m.register_buffer("other", torch.zeros(1))
        m.register_parameter("more", torch.nn.Parameter(torch.zeros(1)))
        m.register_full_backward_hook(lambda *a: None)
        m.register_state_dict_post_hook(lambda *a: None)
        m.register_buffer("unsaved", torch.zeros(1), persistent=False)
        m.add_module("extra", torch.nn.Identity())
    x = torch.randn(5, 40, device="cuda")
    with torch.no_grad():
        model(x)
    assert not seen
    assert all("extra" not in k and "other" not in k and "more" not in k and "unsaved" not in k
               for k, _ in [*model.named_modules(), *model.named_buffers(), *model.named_parameters()])
    assert served.factor is model.factor and served[1][0] is model[1][0]
    assert "unsaved" not in model._non_persistent_buffers_set


def test_a_layer_of_degree_0_stays_among_packed_ones():
    model = torch.nn.Sequential(a_layer(), a_layer(24, 12, 0, seed=1), a_layer(12, 8, 2, seed=2))
    served = kan_b200.quantize_int8(model)
    assert served[1] is model[1] and [type(m).__name__ for m in (served[0], served[2])] == ["Int8ChebyKANLayer"] * 2
    x = torch.randn(5, 40, device="cuda")
    with torch.no_grad():
        assert torch.equal(served(x), served[2](model[1](x.new_zeros(5, 24))))       # the constant is the same for every input


def test_forward_hooks_and_mode_of_a_replaced_layer_go_with_it():
    model = torch.nn.Sequential(a_layer(), a_layer(24, 8, seed=1).eval()).cuda()
    seen = []
    handle = model[0].register_forward_hook(lambda m, args, y: seen.append((type(m).__name__, tuple(y.shape))))
    model[1].register_forward_pre_hook(lambda m, args, kwargs: ((args[0] * 0,), kwargs), with_kwargs=True)
    model[1].register_forward_hook(lambda m, args, kwargs, y: y + 1, with_kwargs=True, always_call=True)
    served = kan_b200.quantize_int8(model)
    assert [m.training for m in served] == [True, False]
    x = torch.randn(5, 40, device="cuda")
    with torch.no_grad():
        y = served(x)
        assert seen == [("Int8ChebyKANLayer", (5, 24))]
        plain = kan_b200.Int8ChebyKANLayer(model[1])
        assert torch.equal(y, plain(torch.zeros(5, 24, device="cuda")) + 1)
        handle.remove()                                  # the original's; the served layer has its own copy
        model(x)
        served(x)
    assert len(seen) == 2


def test_a_module_used_twice_stays_one_module():
    layer = a_layer(24, 24)
    block = torch.nn.Sequential(torch.nn.LayerNorm(24), layer).cuda()
    model = torch.nn.Sequential(a_layer(), block, layer, block)
    served = kan_b200.quantize_int8(model)
    assert served[1] is served[3] and served[1][1] is served[2] and served[1] is not block
    packed = [m for m in served.modules() if isinstance(m, kan_b200.Int8ChebyKANLayer)]
    assert len(packed) == 2 and len(list(served.modules())) == len(list(model.modules()))
    x = torch.randn(5, 40, device="cuda")
    with torch.no_grad():
        y = served[0](x)
        for m in (block[0], packed[1], packed[1], block[0], packed[1]):
            y = m(y)
        assert torch.equal(served(x), y)


def test_buffers_of_the_caller_are_cast():
    layer = kan_b200.quantize_int8(a_layer())
    layer.register_buffer("offset", torch.ones(24, device="cuda"))
    layer.register_buffer("nothing", None)
    layer.half()
    assert layer.offset.dtype == torch.float16 and layer.nothing is None and layer.w_scale.dtype == torch.float32
    assert layer(torch.randn(3, 40, device="cuda")).shape == (3, 24)


def pruned(layer):
    torch.nn.utils.prune.random_unstructured(layer, "cheby_coeffs", 0.5)


def normalised(layer):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        torch.nn.utils.weight_norm(layer, "cheby_coeffs")


def parametrised(layer):
    torch.nn.utils.parametrize.register_parametrization(layer, "cheby_coeffs", torch.nn.Tanh())


@pytest.mark.parametrize("change", [pruned, normalised, parametrised])
def test_a_layer_whose_coefficients_are_rebuilt_is_packed_as_it_stands(change):
    layer = a_layer()
    change(layer)
    seen = []
    layer.register_forward_pre_hook(lambda m, args: seen.append(1))
    x = torch.randn(9, 40, device="cuda")
    with torch.no_grad():
        full = layer(x)
        served = kan_b200.quantize_int8(torch.nn.Sequential(layer))
        y = served(x)
        assert len(seen) == 2 and torch.equal(y, kan_b200.Int8ChebyKANLayer(layer)(x))
        # a basis value is off by half a step of 1/127, a coefficient by half a step of its output's largest: about one percent
        assert float((y - full).norm() / full.norm()) <= 2e-2
