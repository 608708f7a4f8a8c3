"""Newton-Schulz orthogonalisation and the Muon update against the same formulas in 64 bits.

Tolerances.  A step multiplies three times; the quintic's slope stays below 4 where singular values have settled, and
errors of different steps are independent.  Operands of 11 bits (u = 2^-11 at most, u / sqrt(3) in the mean square):
4 * sqrt(15) * 2^-11 / sqrt(3) = 4.4e-3.  Operands of 22 bits: 2.2e-6, plus fp32 sums; the library's fp32 tolerance of
1e-5 is kept.  A result rounded to bf16 adds 2^-8 / sqrt(3) = 2.3e-3 at most, to fp16 2^-11 / sqrt(3) = 2.9e-4."""
import pytest
import torch

import kan_b200
from kan_b200 import graph, ops, optim
from _util import FP32_TOL, assert_guards_intact, guarded

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
TOL = {("fp32x3", torch.float32): FP32_TOL, ("tf32", torch.float32): 4.4e-3,
       ("fp32x3", torch.float16): FP32_TOL + 2.9e-4, ("tf32", torch.float16): 4.4e-3 + 2.9e-4,
       ("fp32x3", torch.bfloat16): FP32_TOL + 2.3e-3, ("tf32", torch.bfloat16): 4.4e-3 + 2.3e-3}


def ns64(g, steps=5, coef=COEF, eps=1e-7):
    x = g.double()
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        a = x @ x.mT
        x = coef[0] * x + (coef[1] * a + coef[2] * a @ a) @ x
    return x.mT if tall else x


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


SHAPES = [(1, 1, 1), (1, 1, 37), (1, 37, 1), (2, 3, 5), (1, 10, 64), (33, 64, 64), (5, 784, 64), (3, 127, 129), (2, 128, 128), (2, 113, 2048), (2, 1300, 97), (40, 50, 400),
          (1, 129, 257), (3, 777, 1000), (1, 20, 5000), (2, 3000, 100), (1, 1, 5000), (2, 256, 1100), (1, 1024, 1024), (1, 2048, 640)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("mode", ["fp32x3", "tf32"])
def test_orthogonalize(shape, mode):
    g = randn(*shape, seed=1, scale=1e-3)
    o = ops.orthogonalize(g, mode=mode)
    assert o.shape == g.shape and o.dtype == g.dtype and o.is_contiguous()
    assert rel(o, ns64(g)) <= TOL[mode, torch.float32]
    assert torch.equal(o, ops.orthogonalize(g, mode=mode))            # repeatable bit for bit
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 3, 5), (3, 130, 70), (1, 300, 520)])
def test_orthogonalize_16_bit(shape, dtype):
    g = randn(*shape, seed=2, dtype=dtype)
    want = ns64(g)
    for mode in (None, "fp32x3", "tf32"):
        used = mode or ("tf32" if dtype == torch.bfloat16 else "fp32x3")
        assert rel(ops.orthogonalize(g, mode=mode), want) <= TOL[used, dtype]


def test_orthogonalize_strides_and_streams():
    base = randn(48, 72, 5, seed=3)
    want = ns64(base.permute(2, 0, 1))
    assert rel(ops.orthogonalize(base.permute(2, 0, 1)), want) <= FP32_TOL          # degree slices of coefficients
    assert rel(ops.orthogonalize(base.permute(2, 1, 0)), want.mT) <= FP32_TOL
    sliced = randn(90, 120, seed=4)[3:80:2, 1:100]                                  # odd offsets, a row stride
    assert rel(ops.orthogonalize(sliced), ns64(sliced)) <= FP32_TOL
    expanded = randn(1, 30, 20, seed=5).expand(4, 30, 20)                           # a batch stride of zero
    assert rel(ops.orthogonalize(expanded), ns64(expanded)) <= FP32_TOL
    side = torch.cuda.Stream()
    g = randn(300, 200, seed=6)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = ops.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    assert rel(o, ns64(g)) <= FP32_TOL


def test_orthogonalize_writes_its_output_only():
    for shape in [(5, 7), (3, 130, 257)]:
        g = randn(*shape, seed=7)
        view, whole = guarded(shape)
        ops.orthogonalize(g, out=view)
        torch.cuda.synchronize()
        assert_guards_intact(view, whole)
        assert rel(view, ns64(g)) <= FP32_TOL


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e30])
def test_orthogonalize_any_magnitude(scale):
    g = randn(2, 70, 90, seed=8, scale=scale)
    # squares of such entries leave fp32; below eps the norm is clamped, as in the definition
    assert rel(ops.orthogonalize(g, eps=1e-35), ns64(g, eps=1e-35)) <= FP32_TOL
    if scale < 1e-12:
        o = ops.orthogonalize(g)
        assert rel(o, ns64(g)) <= FP32_TOL and float(o.abs().max()) < 1e-3


def test_orthogonalize_special_matrices():
    g = randn(5, 40, 60, seed=9)
    g[0] = 0
    g[1, 3, 4] = float("nan")
    g[2, 39, 59] = float("inf")
    g[3, 1:] = 0                                                                   # rank one
    o = ops.orthogonalize(g)
    want = ns64(g[[3, 4]])
    assert bool((o[0] == 0).all()) and bool(torch.isnan(o[1:3]).all())
    assert rel(o[3], want[0]) <= FP32_TOL and rel(o[4], want[1]) <= FP32_TOL
    assert ops.orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert ops.orthogonalize(torch.empty(4, 0, device="cuda")).shape == (4, 0)


@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, COEF), (8, COEF), (6, (2.0, -1.5, 0.5)), (3, (1.5, -0.5, 0.0))])
def test_orthogonalize_steps_and_coefficients(steps, coef):
    g = randn(100, 180, seed=10)
    assert rel(ops.orthogonalize(g, steps=steps, coefficients=coef), ns64(g, steps, coef)) <= FP32_TOL


def muon64(p, g, m, lr, wd, mu, nesterov, scale, gs=1.0):
    g = g.double() * gs
    m = mu * m.double() + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    o = ns64(u.movedim(2, 0)).movedim(0, 2) if u.dim() == 3 else ns64(u)
    return p.double() * (1 - lr * wd) - lr * scale * o, m


@pytest.mark.parametrize("shape", [(1, 1, 9), (64, 64, 33), (784, 64, 5), (64, 10, 5), (130, 257, 3), (48, 96, 128), (300, 200), (512, 512, 2)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(shape, nesterov):
    p, g, m = (randn(*shape, seed=s, scale=sc) for s, sc in ((11, 0.01), (12, 1e-4), (13, 1e-4)))
    rows, cols = (shape[1], shape[0]) if len(shape) == 3 else shape
    want = muon64(p, g, m, 0.5, 0.1, 0.95, nesterov, max(1.0, rows / cols) ** 0.5, 0.25)
    ops.muon_step(p, g, m, lr=0.5, weight_decay=0.1, nesterov=nesterov, grad_scale=0.25)
    assert rel(p, want[0]) <= FP32_TOL and rel(m, want[1]) <= 1e-6
    ops.check_status()


def test_muon_step_writes_its_tensors_only():
    shape = (33, 50, 4)
    g = randn(*shape, seed=14)
    (p, pw), (m, mw) = guarded(shape), guarded(shape)
    p.copy_(randn(*shape, seed=15)); m.zero_()
    want = muon64(p, g, m, 0.5, 0.1, 0.9, True, (50 / 33) ** 0.5)
    ops.muon_step(p, g, m, lr=0.5, momentum=0.9)
    torch.cuda.synchronize()
    assert_guards_intact(p, pw), assert_guards_intact(m, mw)
    assert rel(p, want[0]) <= FP32_TOL and rel(m, want[1]) <= 1e-6


@pytest.mark.parametrize("mode,tol", [("fp32x3", 1e-5), ("tf32", 4.4e-3)])
def test_muon_optimizer_trajectory(mode, tol):
    # five steps on given gradients, of two parameters: the state lives in the optimizer
    params = [torch.nn.Parameter(randn(40, 56, 4, seed=16, scale=0.01)), torch.nn.Parameter(randn(96, 32, seed=17, scale=0.01))]
    opt = optim.Muon(params, lr=0.1, adjust_lr_fn="match_rms_adamw", math_mode=mode)
    want = [(p.detach().double(), torch.zeros_like(p, dtype=torch.float64)) for p in params]
    scales = [0.2 * 56 ** 0.5, 0.2 * 96 ** 0.5]
    for k in range(5):
        for i, p in enumerate(params):
            p.grad = randn(*p.shape, seed=100 * k + i)
            want[i] = muon64(want[i][0], p.grad, want[i][1], 0.1, 0.1, 0.95, True, scales[i])
        versions = [p._version for p in params]
        opt.step()
        assert all(p._version > v for p, v in zip(params, versions))
    for p, (w, _) in zip(params, want):
        assert rel(p.detach(), w) <= tol


def test_muon_graphed_training_step_matches_the_eager_one():
    def model():
        torch.manual_seed(0)
        return torch.nn.Sequential(kan_b200.ChebyKANLayer(12, 24, 4), kan_b200.ChebyKANLayer(24, 8, 4)).cuda()

    x, t = randn(256, 12, seed=18), randn(256, 8, seed=19)
    a, b = model(), model()
    opt_a, opt_b = (optim.Muon(m.parameters(), lr=0.02) for m in (a, b))
    step = graph.GraphedTrainStep(b, kan_b200.mse_loss, opt_b, x, t, warmup=2)
    for _ in range(4):
        step()
    for _ in range(2 + 4):
        opt_a.zero_grad(set_to_none=True)
        kan_b200.mse_loss(a(x), t).backward()
        opt_a.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
    step.close()
    ops.check_status()


@pytest.mark.parametrize("shape", [(2, 300, 520), (3, 60, 900)])
def test_orthogonalize_captured_and_replayed(shape):
    a, b = randn(*shape, seed=20), randn(*shape, seed=21)
    want = [ops.orthogonalize(a), ops.orthogonalize(b)]
    static = a.clone()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:                                   # two graphs that live side by side
        with torch.cuda.graph(g):
            outs.append(ops.orthogonalize(static))
    graphs[0].replay()
    graphs[1].replay()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[0])
    static.copy_(b)
    graphs[1].replay()
    graphs[0].replay()
    assert torch.equal(outs[0], want[1]) and torch.equal(outs[1], want[1])


def test_calls_on_two_streams_at_once():
    inputs = [randn(2, 400, 700, seed=s) for s in range(4)] + [randn(5, 50, 600, seed=s) for s in range(4)]
    want = [ops.orthogonalize(g) for g in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = {}
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for turn in range(3):
        for i, g in enumerate(inputs):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got[i, turn] = ops.orthogonalize(g)
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for (i, _), o in got.items())
    ops.check_status()


def test_muon_step_of_a_large_tensor_in_a_graph():
    shape = (200, 260, 3)
    p, g, m = randn(*shape, seed=22, scale=0.01), randn(*shape, seed=23), randn(*shape, seed=24)
    q, n = p.clone(), m.clone()
    ops.muon_step(p.clone(), g, m.clone(), lr=0.1)
    torch.cuda.synchronize()
    graph_ = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph_):
        ops.muon_step(p, g, m, lr=0.1)
    for _ in range(3):
        graph_.replay()
        ops.muon_step(q, g, n, lr=0.1)
    assert torch.equal(p, q) and torch.equal(m, n)


def test_every_degree_count_of_the_turning_kernels():
    # deg + 1 from 1 to 128 through the tiles that turn [in*out][deg+1] into planes, with a ragged last tile
    for dp1 in (1, 2, 3, 7, 8, 16, 31, 32, 33, 40, 41, 64, 65, 100, 127, 128):
        shape = (9, 11, dp1)
        p, g, m = randn(*shape, seed=25, scale=0.01), randn(*shape, seed=26), randn(*shape, seed=27)
        want = muon64(p, g, m, 0.5, 0.1, 0.95, True, (11 / 9) ** 0.5)
        ops.muon_step(p, g, m, lr=0.5)
        assert rel(p, want[0]) <= FP32_TOL and rel(m, want[1]) <= 1e-6, dp1
