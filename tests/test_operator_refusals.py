"""What the Muon and 8-bit entry points refuse, without a GPU: argument checks come before any device call."""
import pytest
import torch

import kan_b200
from kan_b200 import _lib, ops, optim

P = 4096      # a non-null, aligned stand-in for a device pointer: refused calls read nothing


@pytest.fixture(scope="module")
def lib(built_lib):
    return _lib.load()


def test_workspace_queries(lib):
    x3, tf32 = _lib.MODE_FP32X3, _lib.MODE_TF32
    assert lib.chebykan_orthogonalize_workspace_bytes(1, 640, 640, x3) > lib.chebykan_orthogonalize_workspace_bytes(1, 640, 640, tf32) > 0
    assert lib.chebykan_orthogonalize_workspace_bytes(3, 2048, 128, x3) == 0        # small matrices stay on chip
    assert lib.chebykan_orthogonalize_workspace_bytes(1, 64, 64, _lib.MODE_BF16) == -3
    assert lib.chebykan_orthogonalize_workspace_bytes(1, 64, 64, 9) == -1
    assert lib.chebykan_orthogonalize_workspace_bytes(1, 65537, 64, x3) == -1
    assert lib.chebykan_orthogonalize_workspace_bytes(65536, 64, 64, x3) == -1
    assert lib.chebykan_muon_workspace_bytes(640, 640, 32, x3) > 0
    assert lib.chebykan_muon_workspace_bytes(64, 64, 128, x3) == -1
    assert lib.chebykan_muon_workspace_bytes(0, 64, 4, x3) == -1
    assert lib.chebykan_int8_matmul_workspace_bytes(5, 6, 131072, 131072, 131072) == -1      # the sum could overflow
    assert lib.chebykan_int8_matmul_workspace_bytes(5, 6, 100, 99, 100) == -1                # rows would overlap
    assert lib.chebykan_int8_matmul_workspace_bytes(5, 0, 100, 100, 100) == -1
    assert lib.chebykan_int8_fwd_workspace_bytes(5, 64, 64, 0) == -1                          # degree 0: nothing to quantise
    assert lib.chebykan_int8_fwd_workspace_bytes(5, 2048, 64, 64) == -1                       # 2048 * 64 > 131071
    assert lib.chebykan_int8_fwd_workspace_bytes(50, 64, 64, 4) >= 50 * 256
    assert lib.chebykan_int8_fwd_workspace_bytes(1, 2048, 64, 4) == 0        # a few rows: one launch without a workspace


def orth(lib, **kw):
    a = dict(g=P, sb=0, sr=64, sc=1, dtype=0, out=P, ws=P, ws_bytes=1 << 40, batch=1, m=640, n=640, steps=5, a=3.4445, b=-4.775,
             c=2.0315, eps=1e-7, mode=_lib.MODE_FP32X3, status=P, stream=None)
    a.update(kw)
    return lib.chebykan_orthogonalize(*a.values())


def test_orthogonalize_refuses(lib):
    for kw in (dict(sr=-1), dict(dtype=3), dict(steps=0), dict(steps=33), dict(eps=0.0), dict(eps=float("nan")), dict(g=None), dict(out=None),
               dict(status=None), dict(mode=9), dict(batch=-1)):
        assert orth(lib, **kw) == -1, kw
    # coefficients under which singular values grow without bound, or are no numbers
    assert orth(lib, a=30.0) == -1 and orth(lib, a=float("nan")) == -1 and orth(lib, c=float("inf")) == -1
    assert orth(lib, mode=_lib.MODE_FP32) == -3
    assert orth(lib, out=P + 4) == -2 and orth(lib, ws=P + 8) == -2
    assert orth(lib, ws_bytes=100) == -6 and orth(lib, ws=None) == -6
    assert orth(lib, batch=0) == 0 and orth(lib, m=0, g=None) == 0


def muon(lib, **kw):
    a = dict(param=P, grad=P, buf=P, ws=P, ws_bytes=1 << 40, n_in=640, n_out=640, deg=4, lr=0.1, wd=0.1, mu=0.95, nesterov=1, scale=1.0,
             steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, gs=1.0, mode=_lib.MODE_FP32X3, status=P, stream=None)
    a.update(kw)
    return lib.chebykan_muon_step(*a.values())


def test_muon_step_refuses(lib):
    for kw in (dict(param=None), dict(grad=None), dict(buf=None), dict(status=None), dict(deg=-1), dict(deg=128), dict(n_in=0),
               dict(mu=1.0), dict(mu=-0.1), dict(mu=float("nan")), dict(steps=0), dict(eps=-1.0), dict(b=40.0)):
        assert muon(lib, **kw) == -1, kw
    assert muon(lib, mode=_lib.MODE_BF16) == -3
    assert muon(lib, grad=P + 4) == -2
    assert muon(lib, ws_bytes=100) == -6 and muon(lib, ws=None) == -6


def test_int8_refuses(lib):
    def mm(**kw):
        a = dict(q=P, ldq=64, qs=P, wq=P, ldw=64, ws_=P, bias=None, y=P, dtype=0, ws=P, ws_bytes=1 << 40, M=5, N=6, K=64, status=P, stream=None)
        a.update(kw)
        return lib.chebykan_int8_matmul(*a.values())

    for kw in (dict(q=None), dict(wq=None), dict(qs=None), dict(ws_=None), dict(y=None), dict(status=None), dict(dtype=5), dict(N=0), dict(M=-1),
               dict(K=131072, ldq=131072, ldw=131072), dict(ldq=63)):
        assert mm(**kw) == -1, kw
    assert mm(q=P + 1) == -2 and mm(y=P + 4) == -2
    assert mm(M=0) == 0
    assert lib.chebykan_int8_pack_coeffs(P, P, P, P, 64, 64, 0, None) == -1
    assert lib.chebykan_int8_pack_coeffs(P, P + 4, P, P, 64, 64, 4, None) == -2
    assert lib.chebykan_int8_basis(P, 7, P, P, 5, 64, 4, None) == -1
    assert lib.chebykan_int8_basis(None, 0, P, P, 0, 64, 4, None) == 0
    assert lib.chebykan_int8_fwd(P, 0, P, P, P, P, 0, P, 10, 50, 64, 64, 4, P, None) == -6
    assert lib.chebykan_int8_fwd(P, 0, P, P, P, P, 0, None, 1 << 30, 50, 64, 64, 4, P, None) == -6
    assert lib.chebykan_int8_fwd(P, 0, P, P, P, P, 9, P, 1 << 30, 5, 64, 64, 4, P, None) == -1


def test_python_side_refuses():
    cpu = torch.zeros(4, 4)
    for call in (lambda: ops.orthogonalize(cpu), lambda: ops.muon_step(cpu, cpu, cpu, 0.1), lambda: ops.int8_pack_coeffs(torch.zeros(4, 4, 3)),
                 lambda: ops.int8_basis(cpu, 3), lambda: ops.int8_matmul(cpu.to(torch.int8), cpu[0], cpu.to(torch.int8), cpu[0]),
                 lambda: ops.int8_forward(cpu, cpu.to(torch.int8), cpu[0], None, 1)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(TypeError):
        ops.orthogonalize([1.0])
    with pytest.raises(ValueError, match="adjust"):
        ops.muon_scale((4, 5), "rms")
    with pytest.raises(ValueError, match="SGD or Adam"):
        optim.Muon([torch.nn.Parameter(torch.zeros(5))])
    with pytest.raises(ValueError, match="math_mode"):
        optim.Muon([torch.nn.Parameter(torch.zeros(5, 5))], math_mode="bf16")
    with pytest.raises(ValueError, match="momentum"):
        optim.Muon([torch.nn.Parameter(torch.zeros(5, 5))], momentum=1.0)
    with pytest.raises(ValueError, match="empty"):
        optim.Muon([])
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.Muon([torch.nn.Parameter(torch.zeros(5, 5))])
    with pytest.raises(TypeError):
        kan_b200.Int8ChebyKANLayer(torch.nn.Linear(3, 4))
    with pytest.raises(ValueError, match="degree"):
        kan_b200.Int8ChebyKANLayer(kan_b200.ChebyKANLayer(3, 4, 0))
    with pytest.raises(RuntimeError, match="CUDA"):
        kan_b200.quantize_int8(torch.nn.Sequential(kan_b200.ChebyKANLayer(3, 4, 2)))
    plain = torch.nn.Sequential(torch.nn.Linear(3, 3))
    assert kan_b200.quantize_int8(plain) is plain


def test_muon_scale():
    assert ops.muon_scale((100, 400)) == 1.0 and ops.muon_scale((400, 100)) == 2.0
    assert ops.muon_scale((100, 400, 5)) == 2.0 and ops.muon_scale((400, 100, 5)) == 1.0      # outputs are the rows
    assert abs(ops.muon_scale((100, 400, 5), "match_rms_adamw") - 4.0) < 1e-12
