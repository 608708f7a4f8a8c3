"""The 8-bit forward of a Chebyshev layer, its parts, and a model trained with Muon and served in 8 bits."""
import pytest
import torch

import kan_b200
from kan_b200 import ops, optim
from oracle import chebykan_oracle as o
from _util import assert_guards_intact, guarded, make_case

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def product64(q, qs, wq, ws, bias):
    acc = q.double() @ wq.double().t()
    y = acc * torch.outer(qs.double(), ws.double())
    return y if bias is None else y + bias.double()


def check_product(y, q, qs, wq, ws, bias):
    """The integer sum is exact; its conversion and the product with the row scale are rounded to fp32, the last
    multiply-add once more, the result once to its type."""
    want = product64(q, qs, wq, ws, bias)
    terms = product64(q, qs, wq, ws, None).abs()
    bound = 3 * 2.0 ** -24 * terms + (2.0 ** -24 + HALF_STEP[y.dtype]) * want.abs() * 1.01 + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    assert y.shape == want.shape and bool(((y.double() - want).abs() <= bound).all())


def random_int8(rows, cols, gen, low=-127):
    return torch.randint(low, 128, (rows, cols), generator=gen, device="cuda", dtype=torch.int8)


def case(M, N, K, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + M + 7 * N + 13 * K)
    return (random_int8(M, K, gen), torch.rand(M, generator=gen, device="cuda") * 0.01 + 1e-3, random_int8(N, K, gen),
            torch.rand(N, generator=gen, device="cuda") * 1e-3 + 1e-4, torch.randn(N, generator=gen, device="cuda"))


SHAPES = [(1, 1, 1), (1, 5, 16), (1, 1024, 8192), (2, 7, 33), (3, 64, 100), (5, 10, 320), (8, 130, 272), (4, 70, 1000), (6, 90, 2000), (7, 33, 515), (16, 100, 4096), (17, 65, 64),
          (33, 1, 48), (64, 1000, 256), (100, 129, 1040), (128, 128, 128), (129, 257, 144), (256, 64, 3136), (300, 300, 129),
          (1000, 48, 16), (2000, 10, 64), (1024, 1024, 1024), (5000, 513, 272), (20000, 100, 160), (20000, 20, 400), (9000, 301, 143), (257, 2048, 8192),
          (4, 33, 12288), (4, 33, 12289), (3, 40, 16384), (4, 1300, 2047)]


@pytest.mark.parametrize("shape", SHAPES)
def test_matmul(shape):
    q, qs, wq, ws, bias = case(*shape)
    check_product(ops.int8_matmul(q, qs, wq, ws, bias), q, qs, wq, ws, bias)
    check_product(ops.int8_matmul(q, qs, wq, ws), q, qs, wq, ws, None)
    for dtype in (torch.bfloat16, torch.float16):
        check_product(ops.int8_matmul(q, qs, wq, ws, bias, out_dtype=dtype), q, qs, wq, ws, bias)
    ops.check_status()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_matmul_longest_sum_is_exact(M):
    # K at its limit with every product at its largest: the sum is 131071 * 2^14, just below 2^31
    K, N = 131071, 20
    q = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    wq[1::2] = 127
    one = torch.ones(max(M, N), device="cuda")
    y = ops.int8_matmul(q, one[:M].clone(), wq, one[:N].clone())
    want = torch.tensor([131071.0 * 16384, -131071.0 * 128 * 127] * (N // 2), device="cuda")
    assert torch.equal(y, want.float().expand(M, N))


@pytest.mark.parametrize("M", [1, 4, 7, 200])
def test_matmul_strided_rows_offsets_and_guards(M):
    gen = torch.Generator(device="cuda").manual_seed(M)
    for K, pitch in [(100, 112), (100, 101), (48, 4096)]:
        q = random_int8(M, pitch, gen)[:, :K]
        wq = random_int8(50, pitch, gen)[:, :K]
        qs, ws = torch.rand(M, device="cuda"), torch.rand(50, device="cuda")
        view, whole = guarded((M, 50))
        ops.int8_matmul(q, qs, wq, ws, out=view)
        torch.cuda.synchronize()
        assert_guards_intact(view, whole)
        check_product(view, q, qs, wq, ws, None)


def test_matmul_scales_pass_through():
    q, qs, wq, ws, bias = case(40, 30, 64, seed=5)
    qs[3] = float("nan"); qs[4] = 0; ws[7] = float("inf"); ws[8] = 0
    y = ops.int8_matmul(q, qs, wq, ws, bias)
    assert bool(torch.isnan(y[3]).all()) and torch.equal(y[4, :7], bias[:7])
    assert bool((~torch.isfinite(y[:, 7])).all()) and torch.equal(y[0, 8:9], bias[8:9])
    assert ops.int8_matmul(q[:0], qs[:0], wq, ws, bias).shape == (0, 30)
    assert torch.equal(ops.int8_matmul(q[:, :0], qs.nan_to_num(), wq[:, :0], ws.nan_to_num(posinf=1.0), bias), bias.expand(40, 30))


def exact_basis(x, degree):
    t = torch.tanh(x.double())
    rows, before, here = [t], torch.ones_like(t), t
    for _ in range(degree - 1):
        before, here = here, 2 * t * here - before
        rows.append(here)
    return torch.stack(rows, 1)


@pytest.mark.parametrize("B,n_in,degree", [(1, 1, 1), (3, 1, 8), (5, 17, 3), (300, 64, 32), (9, 255, 4), (9, 257, 4), (257, 784, 4), (40, 2048, 2),
                                           (7, 5000, 6), (33, 16, 127)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_basis(B, n_in, degree, dtype):
    gen = torch.Generator(device="cuda").manual_seed(B + n_in + degree)
    x = (torch.randn(B, n_in, generator=gen, device="cuda") * 1.5).to(dtype)
    x[0] *= 1e-3                                        # a row whose largest value is small (degree 1)
    q, scale = ops.int8_basis(x, degree)
    T = exact_basis(x, degree)
    s = T.abs().amax(dim=(1, 2)) / 127
    # fp32 values of T_d are off by at most (d^2 + 1) 2^-22 of their row's largest: tanh to 2^-22, whose error T_d' <= d^2
    # multiplies, and the recurrence's own roundings, which grow no faster.  A quotient moves by 127 times that, and a
    # rounded one by at most a half more.
    off = (degree ** 2 + 1) * 2.0 ** -22
    assert bool(((scale.double() - s).abs() <= s * off).all())
    q = q.view(B, degree, -1)
    assert q.shape[2] == -(-n_in // 16) * 16 and bool((q[:, :, n_in:] == 0).all())
    assert float((q[:, :, :n_in].double() - T / s[:, None, None]).abs().max()) <= 0.5 + 2 * 127 * off


def test_basis_special_rows():
    x = torch.randn(4, 50, device="cuda")
    x[1, 7] = float("nan"); x[2, 3] = float("inf"); x[2, 4] = -float("inf"); x[3] = 0
    q, scale = ops.int8_basis(x, 1)
    assert bool(torch.isnan(scale[1])) and bool((q[1] == 0).all())
    assert float(scale[2]) == pytest.approx(1 / 127, rel=1e-6) and q[2, 3] == 127 and q[2, 4] == -127
    assert float(scale[3]) == 0 and bool((q[3] == 0).all())
    assert ops.int8_basis(x[:0], 3)[0].shape == (0, 192)


@pytest.mark.parametrize("n_in,n_out,degree", [(1, 1, 1), (17, 5, 3), (784, 64, 4), (300, 129, 8)])
def test_pack(n_in, n_out, degree):
    _, c, _ = make_case(1, n_in, n_out, degree, seed=3)
    c[:, 0, 1:] = 0
    wq, ws, bias = (t.cpu() for t in ops.int8_pack_coeffs(c.cuda()))
    want_s = c[:, :, 1:].abs().amax(dim=(0, 2)) / 127
    assert torch.equal(ws, want_s)
    want = (c[:, :, 1:].permute(1, 2, 0) / want_s.clamp(min=1e-38)[:, None, None]).round()
    wq = wq.view(n_out, degree, -1)
    assert torch.equal(wq[:, :, :n_in].float(), want) and bool((wq[:, :, n_in:] == 0).all())
    assert torch.allclose(bias.double(), c[:, :, 0].double().sum(0), rtol=2.0 ** -23, atol=1e-30)


@pytest.mark.parametrize("B,n_in,n_out,degree", [(1, 2048, 2048, 4), (1, 1, 1, 8), (5, 64, 10, 4), (257, 784, 64, 4), (130, 100, 200, 1),
                                                 (2, 333, 700, 1), (3, 2048, 100, 4), (4, 1000, 3000, 2), (4, 3000, 100, 4),
                                                 (8, 60, 1500, 5), (7, 128, 40, 4), (1000, 64, 64, 32), (700, 1024, 1024, 8)])
def test_forward(B, n_in, n_out, degree):
    x, c, _ = make_case(B, n_in, n_out, degree, seed=4)
    wq, ws, bias = ops.int8_pack_coeffs(c.cuda())
    q, scale = ops.int8_basis(x.cuda(), degree)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = ops.int8_forward(x.cuda(), wq, ws, bias, degree, out_dtype=dtype)
        assert torch.equal(y, ops.int8_matmul(q, scale, wq, ws, bias, out_dtype=dtype))
        check_product(y, q, scale, wq, ws, bias)
    # quantisation: a basis value is off by half a step of 1/127 at most, a coefficient by half a step of its output's
    # largest (about 4 standard deviations) over 127; in the mean square 2.3e-3 and 9e-3 of typical values
    if n_in * degree > 16:
        assert o.rel_l2(ops.int8_forward(x.cuda(), wq, ws, bias, degree).cpu(), o.forward(x, c)) <= 2e-2
    ops.check_status()


@pytest.mark.parametrize("B,n_in,n_out,degree", [(1, 500, 70, 1), (2, 300, 1000, 4), (3, 40, 30, 3), (7, 100, 41, 5)])
def test_forward_of_few_rows_writes_nothing_else_and_keeps_a_nan_to_its_row(B, n_in, n_out, degree):
    gen = torch.Generator(device="cuda").manual_seed(B)
    x = torch.randn(B, n_in, generator=gen, device="cuda")
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(n_in, n_out, degree + 1, generator=gen, device="cuda"))
    for xt in (x.clone(), x.bfloat16(), x.half()):
        view, whole = guarded((B, n_out))
        ops.int8_forward(xt, wq, ws, None, degree, out=view)
        torch.cuda.synchronize()
        assert_guards_intact(view, whole)
        q, scale = ops.int8_basis(xt, degree)
        assert torch.equal(view, ops.int8_matmul(q, scale, wq, ws))
        xt[B - 1, n_in // 2] = float("nan")          # the guard check takes NaN for unwritten
        y = ops.int8_forward(xt, wq, ws, None, degree)
        assert bool(torch.isnan(y[B - 1]).all()) and torch.equal(y[:B - 1], view[:B - 1])


def test_forward_of_more_rows_than_the_workspace_holds():
    # 16 * 127 * 64 = 130048 bytes per quantised row: 8192 rows fill the workspace, the rest is a second turn
    B, n_in, degree = 8500, 1024, 127
    assert ops._lib.load().chebykan_int8_fwd_workspace_bytes(B, n_in, 8, degree) < 1.1e9
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(B, n_in, generator=gen, device="cuda").bfloat16()
    wq = random_int8(8, ops.int8_width(n_in, degree), gen)
    ws = torch.rand(8, generator=gen, device="cuda")
    y = ops.int8_forward(x, wq, ws, None, degree, out_dtype=torch.bfloat16)
    for rows in (slice(0, 40), slice(8180, 8210), slice(8470, 8500)):
        assert torch.equal(y[rows], ops.int8_forward(x[rows].contiguous(), wq, ws, None, degree, out_dtype=torch.bfloat16))


def test_forward_in_a_graph_on_another_stream():
    x, c, _ = make_case(200, 48, 72, 5, seed=6)
    wq, ws, bias = ops.int8_pack_coeffs(c.cuda())
    static = x.cuda()
    want = [ops.int8_forward(static, wq, ws, bias, 5), ops.int8_forward(static.flip(0).contiguous(), wq, ws, bias, 5)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.int8_forward(static, wq, ws, bias, 5)
        z = ops.int8_forward(static, wq, ws, bias, 5, out_dtype=torch.bfloat16)
    g.replay()
    assert torch.equal(y, want[0]) and torch.equal(z, want[0].bfloat16())
    static.copy_(x.cuda().flip(0))
    g.replay()
    assert torch.equal(y, want[1])


def test_train_with_muon_then_serve_in_8_bits():
    torch.manual_seed(0)
    model = torch.nn.Sequential(kan_b200.ChebyKANLayer(8, 32, 5), torch.nn.LayerNorm(32), kan_b200.ChebyKANLayer(32, 4, 5)).cuda()
    kan = [p for p in model.parameters() if p.dim() == 3]
    rest = [p for p in model.parameters() if p.dim() != 3]
    opts = [optim.Muon(kan, lr=0.02), optim.Adam(rest, lr=1e-3)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand(512, 8, generator=gen, device="cuda") * 2 - 1
    t = torch.sin(x @ torch.randn(8, 4, generator=gen, device="cuda"))
    for _ in range(5):
        for opt in opts:
            opt.zero_grad()
        kan_b200.mse_loss(model(x), t).backward()
        for opt in opts:
            opt.step()
    with torch.no_grad():
        full = model(x)
        served = kan_b200.quantize_int8(model)
        assert isinstance(served[0], kan_b200.Int8ChebyKANLayer) and served[1] is model[1] and isinstance(model[0], kan_b200.ChebyKANLayer)
        y = served(x)
        assert y.shape == full.shape and y.dtype == torch.float32
        # two layers of about one percent each; the LayerNorm between them keeps relative errors
        assert float((y - full).norm() / full.norm()) <= 5e-2
        again = kan_b200.Int8ChebyKANLayer(kan_b200.ChebyKANLayer(8, 32, 5).cuda())
        again.load_state_dict(served[0].state_dict())
        assert torch.equal(again(x), served[0](x))
    with pytest.raises(RuntimeError, match="inference"):
        served(x.clone().requires_grad_(True))
    ops.check_status()


def test_matmul_on_two_streams_at_once():
    cases = [case(*s, seed=3) for s in [(300, 500, 640), (20, 64, 4096), (2500, 1100, 300), (1, 700, 999)]]
    want = [ops.int8_matmul(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for turn in range(4):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got.append((i, ops.int8_matmul(*c)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_unaligned_rows_and_half_inputs(dtype):
    # rows of 7 or 13 values start on any 2- or 4-byte boundary
    for B, n_in in [(1, 7), (64, 13), (999, 7), (10, 1001)]:
        x, c, _ = make_case(B, n_in, 21, 3, seed=8)
        x = x.to(dtype).cuda()
        wq, ws, bias = ops.int8_pack_coeffs(c.cuda())
        q, scale = ops.int8_basis(x, 3)
        y = ops.int8_forward(x, wq, ws, bias, 3)
        check_product(y, q, scale, wq, ws, bias)
        assert torch.equal(q, ops.int8_basis(x.float(), 3)[0])         # the type is converted exactly
