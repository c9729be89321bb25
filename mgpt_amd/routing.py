"""ExpertRouting: the choice of experts from a router's logits, and its gradient.

Softmax or sigmoid scores, a bias for balance, groups of experts and
renormalised weights over the C ABI (mgpt_route_forward, mgpt_route_backward,
mgpt_route_balance).  The engine's own router is MoELayer's;
MoELayer.set_routing runs the layer with this one, MoELayer.forward_routed
with a routing that is given.
"""
from __future__ import annotations

import ctypes

import torch

from . import capi

_DT = {"f32": (torch.float32, capi.DTYPE_F32), "bf16": (torch.bfloat16, capi.DTYPE_BF16)}
_SCORE = {"softmax": capi.SCORE_SOFTMAX, "sigmoid": capi.SCORE_SIGMOID}


class ExpertRouting:
    """Logits are [..., E] in `act`'s type.  groups > 1: experts take part by
    groups of E / groups neighbours, the top_groups (None: all) of them whose
    best group_best experts' scores sum to most."""

    def __init__(self, num_experts: int, top_k: int, score: str = "softmax", groups: int = 1,
                 top_groups: int | None = None, group_best: int = 2, renormalise: bool = True, scale: float = 1.0,
                 act: str = "f32"):
        self.E, self.k = num_experts, top_k
        self.dtype, dt = _DT[act]
        self.config = capi.RouteConfig(num_experts, top_k, _SCORE[score], groups,
                                       groups if top_groups is None else top_groups, group_best, int(renormalise),
                                       scale, dt)
        self._cfg = ctypes.byref(self.config)

    @staticmethod
    def _check(t, dtype, shape, device, what):
        if not t.is_cuda or t.device != device:
            raise ValueError(f"{what} must be a CUDA tensor on the device of logits")
        if t.dtype != dtype:
            raise TypeError(f"{what} must be {dtype}")
        if t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous with shape {list(shape)}")
        return t.data_ptr()

    def _logits(self, logits):
        """(address, device, the shape before the experts)"""
        shape, dev = logits.shape, logits.device
        if not shape or shape[-1] != self.E:
            raise ValueError(f"logits must have {self.E} columns")
        return self._check(logits, self.dtype, shape, dev, "logits"), dev, shape[:-1]

    def forward(self, logits, bias=None, counts=None):
        """(idx, weights): int32 and float32 [..., k].  bias: float32 [E], for
        the choice alone.  counts: int32 [E], to which the tokens of each
        expert are added."""
        ptr, dev, rows = self._logits(logits)
        n = capi.rows(rows.numel())
        b = None if bias is None else self._check(bias, torch.float32, (self.E,), dev, "bias")
        c = None if counts is None else self._check(counts, torch.int32, (self.E,), dev, "counts")
        with capi.on_device(dev):
            idx = torch.empty((*rows, self.k), dtype=torch.int32, device=dev)
            weights = torch.empty_like(idx, dtype=torch.float32)
            capi.check(capi.lib().mgpt_route_forward(self._cfg, ptr, b, idx.data_ptr(), weights.data_ptr(), c, n,
                                                     capi.stream(dev)))
        return idx, weights

    def backward(self, logits, idx, weights, dweights, dscores=None):
        """The gradient of logits, in their type, for dweights (float32 [..., k])
        and dscores (float32 [E]: of every token's score of each expert), from
        forward's input and outputs; the choice is taken as given."""
        ptr, dev, rows = self._logits(logits)
        n = capi.rows(rows.numel())
        shape = (*rows, self.k)
        ptrs = [self._check(idx, torch.int32, shape, dev, "idx"),
                self._check(weights, torch.float32, shape, dev, "weights"),
                self._check(dweights, torch.float32, shape, dev, "dweights"),
                None if dscores is None else self._check(dscores, torch.float32, (self.E,), dev, "dscores")]
        with capi.on_device(dev):
            dlogits = torch.empty_like(logits)
            capi.check(capi.lib().mgpt_route_backward(self._cfg, ptr, *ptrs, dlogits.data_ptr(), n,
                                                      capi.stream(dev)))
        return dlogits

    def balance(self, bias, counts, rate: float) -> None:
        """bias += rate for the experts with fewer tokens in counts than the mean,
        -= rate for those with more, in place."""
        if not bias.is_cuda:
            raise ValueError("bias must be a CUDA tensor")
        b = self._check(bias, torch.float32, (self.E,), bias.device, "bias")
        c = self._check(counts, torch.int32, (self.E,), bias.device, "counts")
        with capi.on_device(bias.device):
            capi.check(capi.lib().mgpt_route_balance(self.E, c, rate, b, capi.stream(bias.device)))
