"""Work of the optimizer's and the 8-bit serving path's operators: plain forms, real sizes and 64-bit values.

Four operators on a layer's coefficients:

* ``muon_step``       one Muon update of a coefficient tensor [in, out, degree+1]: momentum, Newton-Schulz
                      orthogonalisation of every degree's in x out matrix, decayed weights and the step;
* ``orthogonalize``   the Newton-Schulz orthogonalisation by itself, on a batch of matrices;
* ``int8_matmul``     y = (q wq^T) * scale[row] * w_scale[column] + bias from 8-bit integers;
* ``int8_forward``    a Chebyshev layer's forward in 8 bits: basis rows quantised per row, then the product.

``run`` computes them in elementary torch operations, or through ``kan_b200`` where ``own`` is set.
"""
import math

import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
LR, DECAY, MOMENTUM = 1e-3, 0.1, 0.95
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    def muon(name, n_in, n_out, degree):
        return {"name": name, "op": "muon_step", "in": n_in, "out": n_out, "degree": degree}

    def orth(name, batch, m, n, dtype):
        return {"name": name, "op": "orthogonalize", "batch": batch, "m": m, "n": n, "dtype": dtype}

    def matmul(name, rows, k, n, dtype):
        return {"name": name, "op": "int8_matmul", "rows": rows, "k": k, "n": n, "dtype": dtype}

    def forward(name, rows, n_in, n_out, degree, dtype):
        return {"name": name, "op": "int8_forward", "rows": rows, "in": n_in, "out": n_out, "degree": degree, "dtype": dtype}

    return [
        # the update of one layer of the narrow degree-32 stack: 33 matrices of 64 x 64
        muon("muon 64x64 degree 32", 64, 64, 32),
        # the update of the 784 -> 64 layer of the image classifier: tall matrices
        muon("muon 784x64 degree 4", 784, 64, 4),
        # the update of the wide layer: nine square matrices, the usual heavy step
        muon("muon 1024x1024 degree 8", 1024, 1024, 8),
        # one matrix of the classifier's 64 -> 10 head: the smallest call, latency alone
        orth("orthogonalize 64x10 f32", 1, 64, 10, "float32"),
        # ragged 16-bit gradients, no size a multiple of a tile
        orth("orthogonalize 3x777x1000 bf16", 3, 777, 1000, "bfloat16"),
        # a degree of each of the four 2048 x 2048 layers of the deep stack, 16-bit gradients
        orth("orthogonalize 4x2048x2048 bf16", 4, 2048, 2048, "bfloat16"),
        # one sample through the wide layer's matrix: bound by reading the 8 MB of weights
        matmul("int8 1x8192 to 1024 f32", 1, 8192, 1024, "float32"),
        # a batch of the classifier through its first layer's matrix: few tiles, a long sum
        matmul("int8 256x3136 to 64 f32", 256, 3136, 64, "float32"),
        # the wide layer's matrix on its full batch
        matmul("int8 65536x8192 to 1024 bf16", 65536, 8192, 1024, "bfloat16"),
        # one sample through one layer of the deep stack
        forward("int8 layer 1x2048 to 2048 d4", 1, 2048, 2048, 4, "bfloat16"),
        # a batch (one row more than a usual 256) of the classifier's first layer
        forward("int8 layer 257x784 to 64 d4", 257, 784, 64, 4, "float16"),
        # one layer of the deep stack on its full batch
        forward("int8 layer 32768x2048 to 2048", 32768, 2048, 2048, 4, "bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["muon_step", "orthogonalize", "int8_matmul", "int8_forward"])
    if op == "muon_step":
        degree = rng.randint(1, 16)
        n_in, n_out = _log(rng, 4, 1200), _log(rng, 4, 1200)
        while n_in * n_out * (degree + 1) > 6_000_000:
            degree = max(1, degree - 1)
            n_in, n_out = max(4, n_in * 4 // 5), max(4, n_out * 4 // 5)
        return {"op": op, "in": n_in, "out": n_out, "degree": degree}
    if op == "orthogonalize":
        return {"op": op, "batch": rng.randint(1, 4), "m": _log(rng, 4, 2048), "n": _log(rng, 4, 2048),
                "dtype": rng.choice(sorted(TYPES))}
    if op == "int8_matmul":
        return {"op": op, "rows": _log(rng, 1, 20000), "k": _log(rng, 8, 8192), "n": _log(rng, 4, 2048),
                "dtype": rng.choice(sorted(TYPES))}
    return {"op": op, "rows": _log(rng, 1, 20000), "in": _log(rng, 2, 1024), "out": _log(rng, 4, 1024),
            "degree": rng.randint(1, 8), "dtype": rng.choice(["bfloat16", "float16"])}


def prepare(case, seed):
    """What a program holds before the call; made on the GPU from the seed."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if op == "muon_step":
        n_in, n_out, dp1 = case["in"], case["out"], case["degree"] + 1
        # the gradient of a layer: basis values of a batch against the gradient of its output
        rows = max(512, 4 * max(n_in, n_out))
        theta = torch.acos(torch.tanh(randn(rows, n_in)))
        dy = randn(rows, n_out) / (rows * n_out)
        grad = torch.empty(n_in, n_out, dp1, device="cuda")
        for d in range(dp1):
            grad[:, :, d] = torch.cos(theta * d).t() @ dy
        std = 1.0 / (n_in * dp1)
        return {"op": op, "param": randn(n_in, n_out, dp1) * std, "grad": grad,
                "buf": 0.5 * grad + randn(n_in, n_out, dp1) * grad.std() * 0.5}
    if op == "orthogonalize":
        g = randn(case["batch"], case["m"], case["n"]) * 1e-3
        return {"op": op, "g": g.to(TYPES[case["dtype"]])}
    if op == "int8_matmul":
        rows, k, n = case["rows"], case["k"], case["n"]
        q = torch.randint(-127, 128, (rows, k), generator=gen, device="cuda", dtype=torch.int8)
        wq = (randn(n, k) * 30).round().clamp(-127, 127).to(torch.int8)
        return {"op": op, "q": q, "scale": torch.rand(rows, generator=gen, device="cuda") * 2e-3 + 6e-3, "wq": wq,
                "w_scale": torch.rand(n, generator=gen, device="cuda") * 1e-4 + 1e-5, "bias": randn(n) * 0.1,
                "dtype": TYPES[case["dtype"]]}
    n_in, n_out, degree = case["in"], case["out"], case["degree"]
    pad = -(-n_in // 16) * 16
    # coefficients in 8 bits: [out][degree 1..D][in], inputs padded with zeros to a multiple of 16, a scale per output
    c = randn(n_out, degree, n_in) / (n_in * (degree + 1))
    w_scale = c.abs().amax(dim=(1, 2)) / 127
    wq = torch.zeros(n_out, degree, pad, dtype=torch.int8, device="cuda")
    wq[:, :, :n_in] = (c / w_scale[:, None, None]).round().to(torch.int8)
    return {"op": op, "x": randn(case["rows"], n_in), "wq": wq.view(n_out, degree * pad), "w_scale": w_scale,
            "bias": randn(n_out) / (degree + 1) / math.sqrt(n_in), "degree": degree, "dtype": TYPES[case["dtype"]]}


def _newton_schulz(u):
    """u[..., m, n] in 32 bits, orthogonalised."""
    tall = u.shape[-2] > u.shape[-1]
    x = u.transpose(-1, -2) if tall else u
    x = x / x.square().sum(dim=(-1, -2), keepdim=True).sqrt().clamp(min=EPS)
    for _ in range(STEPS):
        a = x @ x.transpose(-1, -2)
        x = COEF[0] * x + (COEF[1] * a + COEF[2] * (a @ a)) @ x
    return x.transpose(-1, -2) if tall else x


def run(state):
    op = state["op"]
    if own:
        from kan_b200 import ops
        if op == "muon_step":
            ops.muon_step(state["param"], state["grad"], state["buf"], lr=LR, weight_decay=DECAY, momentum=MOMENTUM)
            return state["param"], state["buf"]
        if op == "orthogonalize":
            return ops.orthogonalize(state["g"])
        if op == "int8_matmul":
            return ops.int8_matmul(state["q"], state["scale"], state["wq"], state["w_scale"], state["bias"],
                                   out_dtype=state["dtype"])
        return ops.int8_forward(state["x"], state["wq"], state["w_scale"], state["bias"], state["degree"],
                                out_dtype=state["dtype"])
    if op == "muon_step":
        param, grad, buf = state["param"], state["grad"], state["buf"]
        buf.add_((grad - buf) * (1 - MOMENTUM))
        u = grad + (buf - grad) * MOMENTUM
        o = _newton_schulz(u.permute(2, 0, 1)).permute(1, 2, 0)
        scale = math.sqrt(max(1.0, param.shape[1] / param.shape[0]))
        param.mul_(1 - LR * DECAY).sub_(o * (LR * scale))
        return param, buf
    if op == "orthogonalize":
        return _newton_schulz(state["g"].float()).to(state["g"].dtype)
    if op == "int8_matmul":
        y = (state["q"].float() @ state["wq"].float().t()) * state["scale"][:, None] * state["w_scale"] + state["bias"]
        return y.to(state["dtype"])
    x, degree = state["x"], state["degree"]
    pad = state["wq"].shape[1] // degree
    # angles and quotients in 64 bits: a value next to a rounding border moves by a whole step
    theta = torch.acos(torch.tanh(x.double()))
    basis = torch.cos(theta[:, None, :] * torch.arange(1, degree + 1, device=x.device)[:, None])
    scale = (basis.abs().amax(dim=(1, 2)) / 127).float()
    q = (basis / scale.double()[:, None, None]).round().float()
    q = torch.nn.functional.pad(q, (0, pad - x.shape[1])).flatten(1)
    y = (q @ state["wq"].float().t()) * scale[:, None] * state["w_scale"] + state["bias"]
    return y.to(state["dtype"])


def work(case):
    op = case["op"]
    if op in ("muon_step", "orthogonalize"):
        m, n = (case["in"], case["out"]) if op == "muon_step" else (case["m"], case["n"])
        s, l = min(m, n), max(m, n)
        # a step: x x^T and a a of which half is enough (both are symmetric), and the product with x
        flops = STEPS * (s * (s + 1) * l + s * s * (s + 1) + 2 * s * s * l)
        if op == "muon_step":    # gradient in; buffer and weights in and out
            return {"bytes": 20 * m * n * (case["degree"] + 1), "flops": flops * (case["degree"] + 1)}
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * size * case["batch"] * m * n, "flops": flops * case["batch"]}
    size = 4 if case["dtype"] == "float32" else 2
    if op == "int8_matmul":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": rows * k + n * k + 4 * (rows + 2 * n) + size * rows * n, "flops": 2 * rows * k * n}
    rows, n_in, n_out, degree = case["rows"], case["in"], case["out"], case["degree"]
    pad = -(-n_in // 16) * 16
    return {"bytes": 4 * rows * n_in + n_out * degree * pad + 8 * n_out + size * rows * n_out,
            "flops": 2 * rows * n_in * degree * n_out}


def exact(case, seed):
    """The outputs of ``run`` from the definitions, in 64 bits; None where the 64-bit product would take too long."""
    op = case["op"]
    s = prepare(case, seed)
    if op in ("muon_step", "orthogonalize"):
        if op == "muon_step":
            g, b = s["grad"].double(), s["buf"].double()
            m = MOMENTUM * b + (1 - MOMENTUM) * g
            z = ((1 - MOMENTUM) * g + MOMENTUM * m).movedim(2, 0)
        else:
            z = s["g"].double()
        z = z / torch.linalg.matrix_norm(z, keepdim=True).clamp_min(EPS)
        wide = z.shape[-1] >= z.shape[-2]
        for _ in range(STEPS):    # x (a + b x^T x + c (x^T x)^2), from the side whose product is smaller
            gram = z @ z.mT if wide else z.mT @ z
            poly = torch.addcmul(COEF[0] * torch.eye(gram.shape[-1], dtype=torch.float64, device=z.device), gram,
                                 torch.full_like(gram, COEF[1])) + COEF[2] * torch.linalg.matrix_power(gram, 2)
            z = poly @ z if wide else z @ poly
        if op == "orthogonalize":
            return z
        factor = LR * max(1.0, case["out"] / case["in"]) ** 0.5
        return s["param"].double() * (1 - LR * DECAY) - factor * z.movedim(0, 2), m
    if 2.0 * s["wq"].numel() * case["rows"] > 1e14:
        return None
    if op == "int8_matmul":
        acc = torch.einsum("mk,nk->mn", s["q"].double(), s["wq"].double())
        return acc * torch.outer(s["scale"].double(), s["w_scale"].double()) + s["bias"].double()
    t = torch.tanh(s["x"].double())
    degrees, before, here = [t], torch.ones_like(t), t
    for _ in range(case["degree"] - 1):
        before, here = here, 2 * t * here - before
        degrees.append(here)
    basis = torch.stack(degrees, 1)
    scale = (basis.abs().flatten(1).max(1).values / 127).float().double()
    q = torch.round(basis / scale.view(-1, 1, 1))
    w = s["wq"].double().view(case["out"], case["degree"], -1)[:, :, :case["in"]]
    return torch.einsum("bdi,odi->bo", q, w) * torch.outer(scale, s["w_scale"].double()) + s["bias"].double()
