"""What the Muon and 8-bit entry points refuse beyond test_operator_refusals.py, without a GPU.  Every call here has to be
refused before a device is asked for: its pointers are stand-ins."""
import pytest

from kan_b200 import _lib
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
