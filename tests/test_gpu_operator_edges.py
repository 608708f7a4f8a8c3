"""Muon, orthogonalisation and 8-bit calls where they could go wrong at the edges: kernels that overlap their predecessor,
tiny and huge values, tensors that are not the plain kind."""
import pytest
import torch

import kan_b200
from kan_b200 import graph, ops, optim
from test_gpu_muon import muon64, randn, rel
from _util import FP32_TOL

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(100, 300, 3), (60, 1001, 2), (7, 2047, 4), (128, 1500), (33, 517, 9)])
def test_muon_step_of_wide_small_matrices_in_a_row(shape):
    # rows lie along memory and their ends fall anywhere in a sector, so the CTAs of a matrix write to shared ones, while the
    # blocks of the update that follows are resident already
    p, g, m = randn(*shape, seed=31, scale=0.01), randn(*shape, seed=32), torch.zeros(shape, device="cuda")
    rows, cols = (shape[1], shape[0]) if len(shape) == 3 else shape
    want, wm = p.double(), m.double()
    for k in range(6):
        g.copy_(randn(*shape, seed=40 + k))
        want, wm = muon64(want, g, wm, 0.5, 0.1, 0.95, True, max(1.0, rows / cols) ** 0.5)
        ops.muon_step(p, g, m, lr=0.5)
    # each step adds an update of at most FP32_TOL relative error to weights that shrink; errors of six add up at most
    assert rel(p, want) <= FP32_TOL * 6 and rel(m, wm) <= 1e-6
    ops.check_status()


@pytest.mark.parametrize("B,n_in,n_out,degree", [(40, 300, 90, 1), (3000, 64, 1100, 1), (20000, 40, 72, 1), (5, 900, 600, 1)])
def test_int8_forward_in_a_row_takes_the_scales_of_its_own_rows(B, n_in, n_out, degree):
    # the workspace is the same memory in every call: a scale left from the call before would show
    gen = torch.Generator(device="cuda").manual_seed(B)
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(n_in, n_out, degree + 1, generator=gen, device="cuda"))
    xs = [torch.randn(B, n_in, generator=gen, device="cuda") * s for s in (1.0, 0.1, 3.0, 0.01)]
    ys = [ops.int8_forward(x, wq, ws, bias, degree) for x in xs]
    for x, y in zip(xs, ys):
        q, scale = ops.int8_basis(x, degree)
        torch.cuda.synchronize()
        assert torch.equal(y, ops.int8_matmul(q, scale, wq, ws, bias))
    ops.check_status()


def test_outputs_beside_their_inputs_are_accepted_and_over_them_refused():
    memory = torch.zeros(6 * 40 * 60, device="cuda")
    parts = [t.view(2, 40, 60) for t in memory.chunk(3)]                # adjacent, nothing between them
    parts[0].copy_(randn(2, 40, 60, seed=50))
    want = ops.orthogonalize(parts[0])
    assert torch.equal(ops.orthogonalize(parts[0], out=parts[1]), want)
    turned = memory.view(-1)[:6 * 40 * 40].view(40, 40, 6).permute(2, 0, 1)
    for g, out in ((parts[0], parts[0]), (turned[:2], parts[0].view(-1)[:3200].view(2, 40, 40)), (turned, memory[4800:].view(-1)[:9600].view(6, 40, 40))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.orthogonalize(g, out=out)
    p, g, m = parts
    m.zero_(); g.copy_(randn(2, 40, 60, seed=51))
    before = p.clone()
    ops.muon_step(p, g, m, lr=0.1)
    assert not torch.equal(p, before)
    for args in ((p, p, m), (p, g, p), (p, g, g)):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.muon_step(*args, lr=0.1)


def test_int8_outputs_over_their_inputs_are_refused():
    x = torch.randn(30, 64, device="cuda")
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(64, 64, 4, device="cuda"))
    q, scale = ops.int8_basis(x, 3)
    for call in (lambda: ops.int8_forward(x, wq, ws, bias, 3, out=x), lambda: ops.int8_forward(x[:2], wq, ws, bias, 3, out=x[1:3]),
                 lambda: ops.int8_matmul(q, scale, wq[:1], ws[:1], bias[:1], out=scale.view(30, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
    memory = torch.empty(60, 64, device="cuda")
    memory[:30] = x
    assert torch.equal(ops.int8_forward(memory[:30], wq, ws, bias, 3, out=memory[30:]), ops.int8_forward(x, wq, ws, bias, 3))


@pytest.mark.parametrize("n_in", [7, 100, 300, 3000, 5000])
def test_int8_basis_of_tiny_rows(n_in):
    # degree 1: tanh x = x for such values, and the scale is a subnormal number from a largest value of 1.5e-36 down
    gen = torch.Generator(device="cuda").manual_seed(n_in)
    tops = [1e-28, 1e-30, 9e-31, 3e-37, 1e-38, 1e-40, 190 * 2.0 ** -149, 64 * 2.0 ** -149, 63 * 2.0 ** -149, 2.0 ** -149]
    x = torch.rand(len(tops), n_in, generator=gen, device="cuda") * 2 - 1
    x[:, 0] = 1
    x[1::2, 0] = -1
    x[:, 2:4] = 0
    x *= 2.0 ** 20                                       # keeps products of small factors exact until the last
    x = (x.double() * torch.tensor(tops, dtype=torch.float64, device="cuda")[:, None] * 2.0 ** -20).float()
    top = x.abs().amax(dim=1)
    q, scale = ops.int8_basis(x, 1)
    assert torch.equal(scale, (top.double() / 127).float())
    want = torch.where(scale[:, None] > 0, x.double() / scale.double()[:, None], 0.0).clamp(-127, 127)
    # the reciprocal of the scale and the quotient are rounded to fp32: 127 * 2^-23, and half a step
    assert float((q[:, :n_in].double() - want).abs().max()) <= 0.5 + 127 * 2.0 ** -23
    assert bool((q[:, 2:4] == 0).all()) and bool((q[:, n_in:] == 0).all())
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(n_in, 20, 2, generator=gen, device="cuda"))
    for rows in (slice(2, 4), slice(0, len(tops))):
        y = ops.int8_forward(x[rows].clone(), wq, ws, None, 1)
        assert torch.equal(y, ops.int8_matmul(q[rows].clone(), scale[rows].clone(), wq, ws)) and bool(torch.isfinite(y).all())


def test_int8_pack_of_the_largest_and_of_no_numbers():
    # finite up to the end of the type; a NaN or an infinity makes its own output NaN
    top = torch.finfo(torch.float32).max
    c = torch.randn(20, 7, 4, device="cuda")
    c[3, 1, 2], c[4, 2, 1], c[5, 3, 3], c[6, 4, 1], c[7, 5, 1:] = top, -3.401e38, float("nan"), -float("inf"), 0
    wq, ws, _ = ops.int8_pack_coeffs(c)
    finite = [0, 1, 2, 5, 6]
    assert torch.equal(ws[finite], (c[:, finite, 1:].abs().amax(dim=(0, 2)).double() / 127).float())
    assert bool(torch.isnan(ws[3:5]).all()) and bool((wq[3:5] == 0).all())
    w = wq.view(7, 3, 32)[:, :, :20].float()
    assert w[1, 1, 3] == 127 and w[2, 0, 4] == -127
    want = c[:, finite, 1:].double().permute(1, 2, 0) / ws[finite].double()[:, None, None]
    # the quotient is rounded to fp32 (2^-24 of up to 127) before it is rounded to an integer
    assert float((w[finite] - want).abs().max()) <= 0.5 + 127 * 2.0 ** -24


class Tagged(torch.Tensor):
    pass


def test_int8_calls_take_tensor_subclasses_and_name_what_is_wrong_with_a_vector():
    x = torch.randn(5, 64, device="cuda")
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(64, 12, 4, device="cuda"))
    q, scale = ops.int8_basis(x, 3)
    want = ops.int8_matmul(q, scale, wq, ws, bias)
    as_tagged = [t.as_subclass(Tagged) for t in (q, scale, wq, ws, bias)]
    assert torch.equal(ops.int8_matmul(*as_tagged).as_subclass(torch.Tensor), want)
    assert torch.equal(ops.int8_forward(x.as_subclass(Tagged), *as_tagged[2:], 3).as_subclass(torch.Tensor), want)
    for bad, words in ((ws[:-1], "12 elements"), (ws.double(), "float32"), (ws.cpu(), "CUDA"), (ws.repeat(2)[::2], "contiguous"),
                       (ws.repeat(2)[1:13], "aligned"), (ws[:-1].as_subclass(Tagged), "12 elements")):
        with pytest.raises(RuntimeError, match=words):
            ops.int8_matmul(q, scale, wq, bad, bias)
        with pytest.raises(RuntimeError, match=words):
            ops.int8_forward(x, wq, ws, bad, 3)


def test_graphed_step_with_muon_for_the_coefficients_and_adam_for_the_rest():
    def parts():
        torch.manual_seed(0)
        model = torch.nn.Sequential(kan_b200.ChebyKANLayer(12, 24, 4), torch.nn.LayerNorm(24), kan_b200.ChebyKANLayer(24, 8, 4)).cuda()
        kan = [p for p in model.parameters() if p.dim() == 3]
        rest = [p for p in model.parameters() if p.dim() != 3]
        return model, [optim.Muon(kan, lr=0.02), optim.Adam(rest, lr=1e-3, capturable=True)]

    x, t = randn(256, 12, seed=18), randn(256, 8, seed=19)
    (a, opts_a), (b, opts_b) = parts(), parts()
    start = [p.detach().clone() for p in a.parameters()]
    step = graph.GraphedTrainStep(b, kan_b200.mse_loss, opts_b, x, t, warmup=2)
    for _ in range(4):
        step()
    for _ in range(2 + 4):
        for opt in opts_a:
            opt.zero_grad(set_to_none=True)
        kan_b200.mse_loss(a(x), t).backward()
        for opt in opts_a:
            opt.step()
    for p, q, was in zip(a.parameters(), b.parameters(), start):
        assert torch.equal(p, q) and not torch.equal(p, was)
    step.close()
    ops.check_status()


@pytest.mark.parametrize("B,n_in,n_out,degree", [(2, 1024, 1000, 4), (2, 1025, 70, 4), (3, 1040, 1000, 8), (4, 1024, 300, 8), (4, 2048, 2048, 4),
                                                 (4, 11000, 40, 1), (1, 11000, 40, 4), (1, 12000, 40, 4), (8, 512, 33, 1), (8, 513, 33, 1)])
def test_int8_forward_on_both_sides_of_one_launch(B, n_in, n_out, degree):
    gen = torch.Generator(device="cuda").manual_seed(B * n_in)
    x = torch.randn(B, n_in, generator=gen, device="cuda")
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(n_in, n_out, degree + 1, generator=gen, device="cuda"))
    for xt in (x, x.half()):
        q, scale = ops.int8_basis(xt, degree)
        for dtype in (torch.float32, torch.bfloat16):
            assert torch.equal(ops.int8_forward(xt, wq, ws, bias, degree, out_dtype=dtype),
                               ops.int8_matmul(q, scale, wq, ws, bias, out_dtype=dtype))
    ops.check_status()
