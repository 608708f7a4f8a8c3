"""What the Muon and 8-bit entry points refuse beyond test_operator_refusals.py, without a GPU.  Every call here has to be
refused before a device is asked for: its pointers are stand-ins."""
import pytest
import torch

import kan_b200
from kan_b200 import _lib, ops, optim
from test_operator_refusals import lib, muon, orth      # noqa: F401  (lib is a fixture)

EOVERLAP = -9
FAR = 1 << 44                                            # out of reach of any tensor here


def test_orthogonalize_refuses_an_output_over_its_input(lib):
    for mode in (_lib.MODE_FP32X3, _lib.MODE_TF32):
        for n in (64, 640):                              # on chip, and through the workspace
            for dtype, size in ((0, 4), (1, 2), (2, 2)):
                kw = dict(m=n, n=n, sr=n, dtype=dtype, mode=mode, ws=2 * FAR)
                assert orth(lib, g=FAR, out=FAR, **kw) == EOVERLAP
                assert orth(lib, g=FAR, out=FAR + size * n * n - 16, **kw) == EOVERLAP
                assert orth(lib, g=FAR + size * n * n - 16, out=FAR, **kw) == EOVERLAP
    # degree slices of coefficients [n, n, 5] against an output over the middle of the same memory
    assert orth(lib, g=FAR, sb=1, sr=5 * 64, sc=5, batch=5, m=64, n=64, out=FAR + 4 * 64 * 64) == EOVERLAP
    assert "overlap" in _lib.strerror(EOVERLAP)


@pytest.mark.parametrize("size", [64, 640])
def test_muon_step_refuses_tensors_over_one_another(lib, size):
    kw = dict(n_in=size, n_out=size, deg=4, ws=5 * FAR)
    last = 4 * size * size * 5 - 16
    for a, b in (("param", "grad"), ("param", "buf"), ("grad", "buf")):
        for by in (0, 16, last):
            tensors = dict(param=FAR, grad=2 * FAR, buf=3 * FAR)
            tensors[b] = tensors[a] + by
            assert muon(lib, **tensors, **kw) == EOVERLAP, (a, b, by)
            tensors[a], tensors[b] = tensors[b], tensors[a]
            assert muon(lib, **tensors, **kw) == EOVERLAP, (b, a, by)


def test_int8_calls_refuse_outputs_over_their_inputs(lib):
    n, k, B = 64, 256, 50

    def matmul(y, q=FAR, qs=2 * FAR, wq=3 * FAR, ws_=4 * FAR, bias=5 * FAR, dtype=0, ldq=k):
        return lib.chebykan_int8_matmul(q, ldq, qs, wq, k, ws_, bias, y, dtype, 7 * FAR, 1 << 30, B, n, k, 4096, None)

    size = {0: 4, 1: 2, 2: 2}
    for dtype in size:
        out = B * n * size[dtype]
        for at, length in ((FAR, B * k), (2 * FAR, 4 * B), (3 * FAR, n * k), (4 * FAR, 4 * n), (5 * FAR, 4 * n)):
            for y in (at, at + (length - 1) // 16 * 16, at - out + 16):
                assert matmul(y, dtype=dtype) == EOVERLAP, (dtype, at, y)
    # rows far apart: the output between them counts as over them
    assert matmul(FAR + 4096, ldq=1 << 20) == EOVERLAP

    def forward(y, rows, x_dtype=0, y_dtype=0):
        return lib.chebykan_int8_fwd(FAR, x_dtype, 3 * FAR, 4 * FAR, 5 * FAR, y, y_dtype, 7 * FAR, 1 << 30, rows, 64, n, 4, 4096, None)

    for rows in (1, B):                                  # one launch, and two
        for xt in size:
            for yt in size:
                out = rows * n * size[yt]
                for at, length in ((FAR, rows * 64 * size[xt]), (3 * FAR, n * k), (4 * FAR, 4 * n), (5 * FAR, 4 * n)):
                    for y in (at, at + (length - 1) // 16 * 16, at - out + 16):
                        assert forward(y, rows, xt, yt) == EOVERLAP, (rows, xt, yt, at, y)
    assert lib.chebykan_int8_basis(FAR, 0, FAR + 4 * B * 64 - 16, 3 * FAR, B, 64, 4, None) == EOVERLAP
    assert lib.chebykan_int8_basis(FAR, 1, 3 * FAR, FAR + 2 * B * 64 - 16, B, 64, 4, None) == EOVERLAP
    for wq, ws_, bias in ((FAR, 3 * FAR, 4 * FAR), (3 * FAR, FAR + 16, 4 * FAR), (3 * FAR, 4 * FAR, FAR + 4 * 64 * n * 5 - 16)):
        assert lib.chebykan_int8_pack_coeffs(FAR, wq, ws_, bias, 64, n, 4, None) == EOVERLAP


def test_int8_forward_never_asks_for_more_than_a_gibibyte(lib):
    for n_in, deg in ((16, 1), (100, 3), (1024, 127), (2000, 65), (16 * 8191, 1)):
        row = -(-n_in // 16) * 16 * deg
        rows = (1 << 30) // row // 256 * 256
        assert rows >= 8192
        for B in (1 << 27, rows + 1, rows):
            assert lib.chebykan_int8_fwd_workspace_bytes(B, n_in, 8, deg) == rows * row + -(-rows * 4 // 256) * 256


def test_operators_without_a_backward_pass_refuse_to_lose_a_gradient():
    t = torch.zeros(16, 16, requires_grad=True)
    q, v = torch.zeros(16, 16, dtype=torch.int8), torch.zeros(16)
    for call in (lambda: ops.orthogonalize(t), lambda: ops.int8_forward(t, q, v, None, 1)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_quantize_int8_leaves_layers_of_degree_0():
    constant = kan_b200.ChebyKANLayer(3, 4, 0)
    model = torch.nn.Sequential(constant, torch.nn.LayerNorm(4))
    assert kan_b200.quantize_int8(constant) is constant and kan_b200.quantize_int8(model) is model


def test_graphed_step_refuses_a_list_with_an_optimizer_that_cannot_be_captured():
    class Fixed:
        capturable = False

    with pytest.raises(ValueError, match="capturable"):
        kan_b200.graph.GraphedTrainStep(torch.nn.Linear(2, 2), kan_b200.mse_loss, [object(), Fixed()], torch.zeros(1, 2), torch.zeros(1, 2))


def test_muon_refuses_its_iteration_when_it_is_made(lib):
    matrix = [torch.nn.Parameter(torch.zeros(5, 5))]
    for kw in (dict(ns_steps=0), dict(ns_steps=33), dict(eps=0.0), dict(eps=-1e-7), dict(eps=float("nan")), dict(ns_coefficients=(30.0, -4.775, 2.0315)),
               dict(ns_coefficients=(float("nan"), 0.0, 0.0))):
        with pytest.raises(ValueError, match="Newton-Schulz"):
            optim.Muon(matrix, **kw)
    for kw in (dict(), dict(ns_steps=32, ns_coefficients=(1.5, -0.5, 0.0)), dict(eps=1e-30)):
        ops.check_newton_schulz(kw.get("ns_steps", 5), kw.get("ns_coefficients", ops.NS_COEFFICIENTS), kw.get("eps", 1e-7))
        with pytest.raises(RuntimeError, match="CUDA"):
            optim.Muon(matrix, **kw)


def test_muon_refuses_shapes_when_it_is_made(lib):
    for shape in ((70000, 1), (1, 70000), (3, 70000, 2), (2, 3, 129)):
        with pytest.raises(ValueError, match="65536"):
            optim.Muon([torch.nn.Parameter(torch.zeros(1).expand(shape))])
        assert lib.chebykan_muon_workspace_bytes(shape[0], shape[1], shape[2] - 1 if len(shape) == 3 else 0, _lib.MODE_FP32X3) == -1
    assert lib.chebykan_muon_workspace_bytes(65536, 2, 127, _lib.MODE_FP32X3) > 0


def test_int8_forward_of_a_few_rows_goes_without_a_workspace_where_one_launch_is_faster(lib):
    def nbytes(B, n_in, deg):
        return lib.chebykan_int8_fwd_workspace_bytes(B, n_in, 64, deg)

    assert all(nbytes(1, n, deg) == 0 for n, deg in ((1, 1), (2048, 4), (4096, 8), (11000, 4)))
    assert all(nbytes(B, n, deg) == 0 for B in (2, 3, 4) for n in (10, 512, 784, 1024) for deg in (1, 4, 8) if B * n * deg <= 46 * 1024)
    assert all(nbytes(B, n, deg) == 0 for B in (5, 8) for n, deg in ((512, 1), (64, 8), (10, 32)))
    # longer rows: two kernels, each quantised once
    assert all(nbytes(B, n, deg) > 0 for B in (2, 3, 4) for n in (1025, 2048, 11000) for deg in (1, 4))
    assert nbytes(1, 12000, 4) > 0 and nbytes(8, 513, 1) > 0 and nbytes(9, 64, 1) > 0
