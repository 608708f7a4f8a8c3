"""Inference with a Chebyshev layer's coefficients in 8 bits.

``quantize_int8`` turns a trained model's ``ChebyKANLayer`` modules into
``Int8ChebyKANLayer``: coefficients of the degrees from 1 in 8-bit integers with
a scale per output, the basis quantised row by row on the way in, an exact
integer product, and the degree-0 term as a bias (``chebykan_int8_fwd``).  A
quarter of the fp32 coefficients' memory; the quantisation error is about one
percent of the output (the rounding of both factors to 8 bits).  Inference only.
"""
from __future__ import annotations

import copy

import torch
import torch.nn as nn

from . import ops


def _is_cheby(m) -> bool:
    return hasattr(m, "cheby_coeffs") and hasattr(m, "math_mode") and hasattr(m, "_packed")


def _packable(m) -> bool:
    return _is_cheby(m) and m.degree > 0


class Int8ChebyKANLayer(nn.Module):
    """8-bit form of a trained ``ChebyKANLayer`` on the GPU; same flatten rule, output in `out_dtype`."""

    def __init__(self, layer: nn.Module, out_dtype: torch.dtype = torch.float32):
        super().__init__()
        if not _is_cheby(layer):
            raise TypeError("Int8ChebyKANLayer is built from a ChebyKANLayer")
        if layer.degree < 1:
            raise ValueError("the 8-bit forward needs a degree of at least 1")
        if not layer.cheby_coeffs.is_cuda:
            raise RuntimeError("move the layer to a CUDA device first: kan_b200 has no CPU path")
        self.input_dim, self.output_dim, self.degree = layer.input_dim, layer.output_dim, layer.degree
        self.out_dtype = out_dtype
        wq, w_scale, bias = ops.int8_pack_coeffs(layer.cheby_coeffs.detach().contiguous())
        self.register_buffer("wq", wq)
        self.register_buffer("w_scale", w_scale)
        self.register_buffer("bias", bias)

    def _apply(self, fn, recurse=True):
        # model.half(), .to(torch.bfloat16), .double(): the kernels take the 8-bit weights, scales and biases as they were
        # packed, whatever type the model around them works in; a move to another device is followed
        packed = {name: self._buffers[name] for name in ("wq", "w_scale", "bias")}
        super()._apply(fn, recurse)
        for name, t in packed.items():
            if self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("the 8-bit layer is for inference: it has no gradient (call it under torch.no_grad())")
        x = x.view(-1, self.input_dim).contiguous()
        if x.numel() and x.data_ptr() % 16:
            x = x.clone()
        return ops.int8_forward(x, self.wq, self.w_scale, self.bias, self.degree, out_dtype=self.out_dtype)

    def extra_repr(self) -> str:
        return f"input_dim={self.input_dim}, output_dim={self.output_dim}, degree={self.degree}"


_MODULE_STATE = [name for name, value in nn.Module().__dict__.items() if isinstance(value, (dict, set))]
_FORWARD_HOOKS = [name for name in _MODULE_STATE if name.startswith(("_forward_hooks", "_forward_pre_hooks"))]


def _rebuilds_coefficients(hook) -> bool:
    return "cheby_coeffs" in (getattr(hook, "_tensor_name", None), getattr(hook, "name", None))


def quantize_int8(model: nn.Module) -> nn.Module:
    """The model with every ``ChebyKANLayer`` in 8 bits; one of degree 0, a constant, stays.  Forward hooks of a replaced layer
    go with it.  Other modules, parameters and buffers are shared with `model`, which stays as it is; casting or moving the
    result reaches what is shared (copy.deepcopy it first)."""
    return _quantized(model, {})


def _quantized(m: nn.Module, done: dict) -> nn.Module:
    """`done`: what became of the modules met so far, so that a module used twice stays one module."""
    if m in done:
        return done[m]
    if _packable(m):
        new = Int8ChebyKANLayer(m)
        new.train(m.training)
        for name in _FORWARD_HOOKS:
            # pruning and weight normalisation hang hooks on a layer that rebuild its coefficients: they are packed already
            new.__dict__[name].update((key, hook) for key, hook in m.__dict__[name].items() if not _rebuilds_coefficients(hook))
    elif any(_packable(c) for c in m.modules()):
        new = copy.copy(m)
        for name in _MODULE_STATE:          # registering a hook, buffer or parameter with the one leaves the other alone
            new.__dict__[name] = copy.copy(m.__dict__[name])
        done[m] = new
        for name, child in m._modules.items():
            new._modules[name] = None if child is None else _quantized(child, done)
    else:
        new = m
    done[m] = new
    return new
