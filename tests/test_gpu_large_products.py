"""The tensor-core products at the sizes where pairs of CTAs take several tiles each: symmetric operands read through mirror
images on both sides, tiles cut in half after the last full wave, accumulators and staging buffers used again.

Errors are compared block by block (128 x 128), so that one wrong tile, or half of one, shows.  The tolerances of
test_gpu_muon.py are statements about single entries (independent roundings), so a block's relative error is the matrix's; a
ragged block has 76 x 104 entries at least, whose mean square error and mean square each stray by a few percent.  1.25 times
the matrix's tolerance covers both."""
import pytest
import torch

from kan_b200 import ops
from test_gpu_int8 import case, check_product, random_int8
from test_gpu_muon import TOL, muon64, ns64, randn

pytestmark = pytest.mark.gpu


def worst_block(got, want, block=128):
    """Largest relative L2 error of a block of the matrices got[..., m, n]."""
    def sums(t):
        t = torch.nn.functional.pad(t, (0, -t.shape[-1] % block, 0, -t.shape[-2] % block))
        return t.unflatten(-1, (-1, block)).unflatten(-3, (-1, block)).square().sum(dim=(-1, -3))

    assert bool(torch.isfinite(got).all())
    return float((sums(got.double() - want) / sums(want)).max().sqrt())


# (9, 1024, 1024): 90 pair tiles with 16 left over for A and P, 144 for X'; (4, 2048, 2048): 144 and 256, so up to four tiles
# per pair, and halves in the last wave of X'; the ragged ones leave halves that lie outside the matrix
@pytest.mark.parametrize("shape", [(9, 1024, 1024), (4, 2048, 2048), (8, 1000, 1100), (8, 1100, 1000), (3, 1400, 2636)])
@pytest.mark.parametrize("mode", ["fp32x3", "tf32"])
def test_orthogonalize(shape, mode):
    g = randn(*shape, seed=1, scale=1e-3)
    o = ops.orthogonalize(g, mode=mode)
    assert worst_block(o, ns64(g)) <= 1.25 * TOL[mode, torch.float32]
    for _ in range(3):
        assert torch.equal(o, ops.orthogonalize(g, mode=mode))
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(4, 2048, 2048), (3, 777, 1000), (6, 1100, 1000)])
def test_orthogonalize_16_bit(shape, dtype):
    g = randn(*shape, seed=2, dtype=dtype, scale=0.1)
    want = ns64(g)
    for mode in (None, "fp32x3"):
        used = mode or ("tf32" if dtype == torch.bfloat16 else "fp32x3")
        o = ops.orthogonalize(g, mode=mode)
        # 777 = 6 * 128 + 9: blocks of as few as 9 x 104 entries, whose error strays by a tenth at four standard deviations
        assert worst_block(o, want) <= 1.25 * TOL[used, dtype]
        assert torch.equal(o, ops.orthogonalize(g, mode=mode))
    ops.check_status()


@pytest.mark.parametrize("shape", [(1024, 1024, 9), (1100, 1000, 8), (1000, 1100, 8), (513, 1300, 17), (1500, 1100)])
@pytest.mark.parametrize("mode", ["fp32x3", "tf32"])
def test_muon_step(shape, mode):
    p, g, m = (randn(*shape, seed=s, scale=sc) for s, sc in ((11, 1e-4), (12, 1e-4), (13, 1e-4)))
    rows, cols = (shape[1], shape[0]) if len(shape) == 3 else shape
    want = muon64(p, g, m, 0.5, 0.1, 0.95, True, max(1.0, rows / cols) ** 0.5)
    q, n = p.clone(), m.clone()
    ops.muon_step(p, g, m, lr=0.5, mode=mode)
    planes = (lambda t: t.movedim(2, 0)) if len(shape) == 3 else (lambda t: t)
    assert worst_block(planes(p), planes(want[0])) <= 1.25 * TOL[mode, torch.float32]
    assert worst_block(planes(m), planes(want[1])) <= 1e-6
    ops.muon_step(q, g, n, lr=0.5, mode=mode)
    assert torch.equal(p, q) and torch.equal(m, n)
    ops.check_status()


# 628 tiles on 74 pairs with 3 and with 1 K block (the MMAs wait for the epilogue), 782 and 391 narrow ones, 316 with 64 K blocks
@pytest.mark.parametrize("shape", [(40000, 1000, 272), (40000, 1000, 16), (100000, 100, 48), (200000, 60, 300), (20000, 1024, 8192), (30001, 1023, 129)])
def test_int8_matmul(shape):
    q, qs, wq, ws, bias = case(*shape, seed=1)
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.int8_matmul(q, qs, wq, ws, bias, out_dtype=dtype)
        check_product(y, q, qs, wq, ws, bias)
        for _ in range(2):
            assert torch.equal(y, ops.int8_matmul(q, qs, wq, ws, bias, out_dtype=dtype))
    ops.check_status()


def test_int8_forward_in_turns_on_the_persistent_product():
    # 130048 bytes per quantised row: 8192 rows per turn, 96 tiles of 256 x 256 each, then a turn of 116 rows
    B, n_in, n_out, degree = 16500, 1024, 700, 127
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(B, n_in, generator=gen, device="cuda").bfloat16()
    wq = random_int8(n_out, ops.int8_width(n_in, degree), gen)
    ws = torch.rand(n_out, generator=gen, device="cuda")
    y = ops.int8_forward(x, wq, ws, None, degree, out_dtype=torch.bfloat16)
    for first in (0, 4000, 8180, 12000, 16300, 16460):
        rows = slice(first, first + 40)
        assert torch.equal(y[rows], ops.int8_forward(x[rows].contiguous(), wq, ws, None, degree, out_dtype=torch.bfloat16))
    ops.check_status()


@pytest.mark.parametrize("degree", [1, 4])
def test_int8_forward_of_a_full_batch(degree):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(32768, 2048, generator=gen, device="cuda")
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(2048, 2048, degree + 1, generator=gen, device="cuda") * 1e-3)
    y = ops.int8_forward(x, wq, ws, bias, degree)
    q, scale = ops.int8_basis(x, degree)
    assert torch.equal(y, ops.int8_matmul(q, scale, wq, ws, bias))
    check_product(y[-3000:], q[-3000:], scale[-3000:], wq, ws, bias)
    assert torch.equal(y, ops.int8_forward(x, wq, ws, bias, degree))
    ops.check_status()


def test_offsets_beyond_32_bits():
    gen = torch.Generator(device="cuda").manual_seed(4)
    # rows of q from byte 2^31 on, on the tensor cores and as a few rows far apart
    q = torch.zeros(270000, 8192, dtype=torch.int8, device="cuda")
    q[-3000:] = random_int8(3000, 8192, gen)
    wq, ws = random_int8(40, 8192, gen), torch.rand(40, generator=gen, device="cuda")
    qs = torch.rand(270000, generator=gen, device="cuda")
    y = ops.int8_matmul(q, qs, wq, ws)
    assert bool((y[:-3000] == 0).all())
    check_product(y[-3000:], q[-3000:], qs[-3000:], wq, ws, None)
    far = q[::269999]
    check_product(ops.int8_matmul(far, qs[:2].clone(), wq, ws), far, qs[:2], wq, ws, None)
    del q, far
    # results from element 2^31 on
    x = torch.randn(2200000, 16, generator=gen, device="cuda")
    wq, ws, bias = ops.int8_pack_coeffs(torch.randn(16, 1000, 3, generator=gen, device="cuda"))
    y = ops.int8_forward(x, wq, ws, bias, 2, out_dtype=torch.bfloat16)
    for first in (0, 1100000, 2147483, 2199000):
        rows = slice(first, first + 1000)
        assert torch.equal(y[rows], ops.int8_forward(x[rows].clone(), wq, ws, bias, 2, out_dtype=torch.bfloat16))
    del x, y
    # matrices 2^31 elements apart, on chip and through the workspace
    memory = torch.zeros(2 ** 31 + 300 * 500, dtype=torch.bfloat16, device="cuda")
    for m, n in ((50, 70), (300, 500)):
        g = memory.as_strided((2, m, n), (2 ** 31, n, 1))
        g.copy_(randn(2, m, n, seed=5))
        assert worst_block(ops.orthogonalize(g, mode="fp32x3"), ns64(g)) <= 1.25 * TOL["fp32x3", torch.bfloat16]
    ops.check_status()
