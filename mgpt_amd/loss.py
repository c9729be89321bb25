"""LMLoss: a language model head's softmax cross entropy without its logits.

Mirrors lm_head (LinearLayer) and CrossEntropyLossLayer of the engine
(/root/reference/src/main/neuralnetwork/layers/CrossEntropyLossLayer.cpp) over
the C ABI (mgpt_lm_loss_forward, mgpt_lm_loss_backward): the forward keeps one
number per token, the backward forms the logits again, a piece of the
vocabulary at a time.
"""
from __future__ import annotations

import ctypes

import torch

from . import capi

_DT = {"f32": (torch.float32, capi.DTYPE_F32), "bf16": (torch.bfloat16, capi.DTYPE_BF16)}


class LMLoss:
    """x [..., C] and weight [V, C] in `act`'s type, bias float32 [V] or None,
    targets int32, one per token; one outside 0 .. V - 1 means that the token
    has none.  The workspace of a call is allocated with torch for that call
    (its stream's, or the captured graph's own)."""

    def __init__(self, embed_dim: int, vocab_size: int, act: str = "bf16"):
        self.C, self.V = embed_dim, vocab_size
        self.dtype, dt = _DT[act]
        self._cfg = capi.LMLossConfig(embed_dim, vocab_size, dt)

    @staticmethod
    def _check(t, dtype, shape, device, what):
        if not t.is_cuda or t.device != device:
            raise ValueError(f"{what} must be a CUDA tensor on the device of x")
        if t.dtype != dtype:
            raise TypeError(f"{what} must be {dtype}")
        if tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous with shape {list(shape)}")
        return t.data_ptr()

    def _inputs(self, x, weight, targets, bias):
        if x.dim() < 1 or x.shape[-1] != self.C:
            raise ValueError(f"x must have {self.C} columns")
        dev = x.device
        ptrs = [self._check(x, self.dtype, tuple(x.shape), dev, "x"),
                self._check(weight, self.dtype, (self.V, self.C), dev, "weight"),
                None if bias is None else self._check(bias, torch.float32, (self.V,), dev, "bias"),
                self._check(targets, torch.int32, tuple(x.shape[:-1]), dev, "targets")]
        return x.numel() // self.C, ptrs

    def _workspace(self, query, n, device):
        need = ctypes.c_size_t()
        capi.check(query(ctypes.byref(self._cfg), n, ctypes.byref(need)))
        return torch.empty(need.value, dtype=torch.uint8, device=device)

    def forward(self, x, weight, targets, bias=None):
        """(loss, lse, mean): per token its loss (0 without a target) and
        log-sum-exp, float32 in the shape of targets, and float32 [2], the mean
        loss over the tokens with a target and their number."""
        n, ptrs = self._inputs(x, weight, targets, bias)
        with capi.on_device(x.device):
            loss = torch.empty(targets.shape, dtype=torch.float32, device=x.device)
            lse = torch.empty_like(loss)
            mean = torch.empty(2, dtype=torch.float32, device=x.device)
            ws = self._workspace(capi.lib().mgpt_lm_loss_workspace_bytes, n, x.device)
            capi.check(capi.lib().mgpt_lm_loss_forward(
                ctypes.byref(self._cfg), *ptrs, loss.data_ptr(), lse.data_ptr(), mean.data_ptr(), n, ws.data_ptr(),
                ws.numel(), capi.stream(x.device)))
        return loss, lse, mean

    def backward(self, x, weight, targets, lse, bias=None, dloss=None, dmean=None, need=(True, True, True)):
        """(dx, dweight, dbias) from forward's inputs and its lse, for the
        upstream gradient dloss (float32, per token) or dmean (float32, one
        element; None: 1) of the mean loss.  need: which of the three are
        wanted; one that is not, and dbias without a bias, is None.  In bf16
        dx and dweight are products of logits' gradients rounded to bf16,
        dbias is their sum before that."""
        n, ptrs = self._inputs(x, weight, targets, bias)
        dev = x.device
        ptrs.append(self._check(lse, torch.float32, tuple(targets.shape), dev, "lse"))
        if dloss is not None and dmean is not None:
            raise ValueError("dloss and dmean exclude each other")
        ptrs.append(None if dloss is None else self._check(dloss, torch.float32, tuple(targets.shape), dev, "dloss"))
        if dmean is not None and dmean.numel() != 1:
            raise ValueError("dmean must have one element")
        ptrs.append(None if dmean is None else self._check(dmean, torch.float32, tuple(dmean.shape), dev, "dmean"))
        with capi.on_device(dev):
            dx = torch.empty_like(x) if need[0] else None
            dw = torch.empty_like(weight) if need[1] else None
            db = torch.empty_like(bias) if need[2] and bias is not None else None
            ws = self._workspace(capi.lib().mgpt_lm_loss_backward_workspace_bytes, n, dev)
            capi.check(capi.lib().mgpt_lm_loss_backward(
                ctypes.byref(self._cfg), *ptrs, *[None if t is None else t.data_ptr() for t in (dx, dw, db)], n,
                ws.data_ptr(), ws.numel(), capi.stream(x.device)))
        return dx, dw, db
