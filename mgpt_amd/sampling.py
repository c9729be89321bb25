"""Sampler: a token for each row of logits from a given random number.

Temperature, top-k, top-p and min-p, for all rows or for each its own, over the
C ABI (mgpt_sample): the sampling of the engine's Generator
(/root/reference/src/main/pipeline/Generator.cpp:13-36) on the device, so
that a decode step needs no copy to the host and can be captured whole.
"""
from __future__ import annotations

import ctypes

import torch

from . import capi

_DT = {"f32": (torch.float32, capi.DTYPE_F32), "bf16": (torch.bfloat16, capi.DTYPE_BF16)}


class Sampler:
    """Logits are [..., V] in `act`'s type.  The workspace of a call is allocated
    with torch for that call (its stream's, or the captured graph's own)."""

    def __init__(self, vocab_size: int, act: str = "f32"):
        self.V = vocab_size
        self.dtype, self._dt = _DT[act]

    @staticmethod
    def _check(t, dtype, shape, device, what):
        if not t.is_cuda or t.device != device:
            raise ValueError(f"{what} must be a CUDA tensor on the device of logits")
        if t.dtype != dtype:
            raise TypeError(f"{what} must be {dtype}")
        if t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous with shape {list(shape)}")
        return t.data_ptr()

    def forward(self, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """(token, logp): int32 and float32 [...], one per row.  u: float32 [...] in
        [0, 1).  temperature (0: the largest logit), top_k (0: all), top_p
        and min_p: numbers, or tensors [...] (int32 for top_k, else float32).
        logp is the token's log-probability among those kept; a row of
        nothing but -inf has token -1."""
        if logits.dim() < 1 or logits.shape[-1] != self.V:
            raise ValueError(f"logits must have {self.V} columns")
        dev, shape = logits.device, logits.shape[:-1]
        n = capi.rows(shape.numel())
        ptr = self._check(logits, self.dtype, logits.shape, dev, "logits")
        up = self._check(u, torch.float32, shape, dev, "u")
        cfg = capi.SampleConfig(self.V, self._dt, 1.0, 0, 1.0, 0.0)
        ptrs = []
        for name, v, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                            ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
            if isinstance(v, torch.Tensor):
                ptrs.append(self._check(v, dt, shape, dev, name))
            else:
                # (32 bits: a top_k past the vocabulary is all of it, as one below 1)
                setattr(cfg, name, max(0, min(v, self.V)) if name == "top_k" else v)
                ptrs.append(None)
        with capi.on_device(dev):
            token = torch.empty(shape, dtype=torch.int32, device=dev)
            logp = torch.empty_like(token, dtype=torch.float32)
            need = ctypes.c_size_t()
            capi.check(capi.lib().mgpt_sample_workspace_bytes(ctypes.byref(cfg), n, ctypes.byref(need)))
            ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
            capi.check(capi.lib().mgpt_sample(ctypes.byref(cfg), ptr, up, *ptrs, token.data_ptr(), logp.data_ptr(),
                                              n, ws.data_ptr(), need.value, capi.stream(dev)))
        return token, logp
