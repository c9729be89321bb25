"""I8Linear: a linear layer in 8-bit integers, a scale for each token and output.

Over the C ABI (mgpt_i8_pack_weight, mgpt_i8_pack_quantized,
mgpt_i8_linear_forward), for serving: the engine's LinearLayer
(/root/reference/src/main/neuralnetwork/layers/LinearLayer.cpp:23-28) with
both operands in int8, as a language model's head.  The experts' form of the
product is MoELayer(weights="i8").
"""
from __future__ import annotations

import ctypes

import torch

from . import capi

_DT = {"f32": (torch.float32, capi.DTYPE_F32), "bf16": (torch.bfloat16, capi.DTYPE_BF16)}


class I8Linear:
    """x [..., K] and the outputs [..., M] are in `act`'s type.  The layer keeps
    the packed weight, its scales and the bias; the workspace of a call is
    allocated with torch for that call."""

    def __init__(self, in_features: int, out_features: int, act: str = "bf16"):
        self.K, self.M = in_features, out_features
        self.dtype, dt = _DT[act]
        self._cfg = capi.I8Config(in_features, out_features, dt)
        self._packed = self.scales = self.bias = None

    def _new(self, weight, bias):
        if not weight.is_cuda:
            raise ValueError("weight must be a CUDA tensor")
        if tuple(weight.shape) != (self.M, self.K) or not weight.is_contiguous():
            raise ValueError(f"weight must be contiguous with shape {[self.M, self.K]}")
        if bias is not None and (bias.device != weight.device or bias.dtype != torch.float32
                                 or tuple(bias.shape) != (self.M,) or not bias.is_contiguous()):
            raise ValueError(f"bias must be a contiguous float32 tensor of {self.M} elements on the weight's device")
        need = ctypes.c_size_t()
        capi.check(capi.lib().mgpt_i8_weight_bytes(ctypes.byref(self._cfg), ctypes.byref(need)))
        return torch.empty(need.value, dtype=torch.uint8, device=weight.device)

    def load(self, weight, bias=None) -> None:
        """weight: float32 or bfloat16 [M, K], quantised here with a scale for each
        row; bias: float32 [M], kept as it is (not copied)."""
        if weight.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("weight must be float32 or bfloat16")
        packed = self._new(weight, bias)
        with capi.on_device(weight.device):
            scales = torch.empty(self.M, dtype=torch.float32, device=weight.device)
            capi.check(capi.lib().mgpt_i8_pack_weight(
                ctypes.byref(self._cfg), weight.data_ptr(),
                capi.DTYPE_F32 if weight.dtype == torch.float32 else capi.DTYPE_BF16, packed.data_ptr(),
                scales.data_ptr(), capi.stream(weight.device)))
        self._packed, self.scales, self.bias = packed, scales, bias

    def load_quantized(self, weight, scales, bias=None) -> None:
        """weight: int8 [M, K] and scales: float32 [M], of which a row's values are
        the product; scales and bias are kept as they are (not copied)."""
        if weight.dtype != torch.int8:
            raise TypeError("weight must be int8")
        packed = self._new(weight, bias)
        if (scales.device != weight.device or scales.dtype != torch.float32 or tuple(scales.shape) != (self.M,)
                or not scales.is_contiguous()):
            raise ValueError(f"scales must be a contiguous float32 tensor of {self.M} elements on the weight's device")
        with capi.on_device(weight.device):
            capi.check(capi.lib().mgpt_i8_pack_quantized(ctypes.byref(self._cfg), weight.data_ptr(),
                                                         packed.data_ptr(), capi.stream(weight.device)))
        self._packed, self.scales, self.bias = packed, scales, bias

    def forward(self, x):
        if self._packed is None:
            raise RuntimeError("no weight has been loaded")
        dev = x.device
        if not x.is_cuda or dev != self._packed.device:
            raise ValueError("x must be a CUDA tensor on the device of the weight")
        if x.dtype != self.dtype:
            raise TypeError(f"x must be {self.dtype}")
        if x.dim() < 1 or x.shape[-1] != self.K or not x.is_contiguous():
            raise ValueError(f"x must be contiguous with {self.K} columns")
        n = capi.rows(x.numel() // self.K)
        with capi.on_device(dev):
            y = torch.empty((*x.shape[:-1], self.M), dtype=self.dtype, device=dev)
            need = ctypes.c_size_t()
            capi.check(capi.lib().mgpt_i8_linear_workspace_bytes(ctypes.byref(self._cfg), n, ctypes.byref(need)))
            ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
            capi.check(capi.lib().mgpt_i8_linear_forward(
                ctypes.byref(self._cfg), x.data_ptr(), self._packed.data_ptr(), self.scales.data_ptr(),
                None if self.bias is None else self.bias.data_ptr(), y.data_ptr(), n, ws.data_ptr(), ws.numel(),
                capi.stream(dev)))
        return y
