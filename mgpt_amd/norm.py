"""ResidualNorm: the norms around a block with its gate and the residual stream.

out = residual_scale * x + gate * (RMSNorm(h) * gamma_post) and
y = RMSNorm(out) * gamma_pre in one pass over x and h, and its backward, over
the C ABI (mgpt_norm_forward, mgpt_norm_backward).  The engine's RMSNormLayer
(/root/reference/src/main/neuralnetwork/layers/RMSNormLayer.cpp) is the
pre-norm alone; MoELayer.forward_block fuses that one into its router.
"""
from __future__ import annotations

import ctypes

import torch

from . import capi

_DT = {"f32": (torch.float32, capi.DTYPE_F32), "bf16": (torch.bfloat16, capi.DTYPE_BF16)}


class ResidualNorm:
    def __init__(self, embed_dim: int, act: str = "bf16", eps: float = 1e-5, residual_scale: float = 1.0):
        self.C = embed_dim
        self.dtype, self._dt = _DT[act]
        self.eps = eps
        self.residual_scale = residual_scale

    def _rows(self, t, shape, device, what):
        if not t.is_cuda or t.device != device:
            raise ValueError(f"{what} must be a CUDA tensor on the device of x")
        if t.dtype != self.dtype:
            raise TypeError(f"{what} must be {self.dtype}")
        if t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous with the shape of x")
        return t.data_ptr()

    def _gains(self, x, gamma_post, gate, gamma_pre):
        """(config, N, the three pointers), checked."""
        if x.dim() < 1 or x.shape[-1] != self.C:
            raise ValueError(f"x must have {self.C} columns")
        n = x.numel() // self.C
        rows = 1
        ptrs = []
        for t, what in ((gamma_post, "gamma_post"), (gate, "gate"), (gamma_pre, "gamma_pre")):
            if t is None:
                ptrs.append(None)
                continue
            if t.device != x.device or t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError(f"{what} must be a contiguous float32 tensor on the device of x")
            if what == "gate":
                if t.dim() < 1 or t.shape[-1] != self.C:
                    raise ValueError(f"gate must have {self.C} columns")
                rows = t.numel() // self.C
                if rows < 1 or n % rows:
                    raise ValueError(f"the gate's {rows} rows must divide the {n} tokens")
            elif t.numel() != self.C:
                raise ValueError(f"{what} must have {self.C} elements")
            ptrs.append(t.data_ptr())
        return capi.NormConfig(self.C, self._dt, rows, self.eps, self.residual_scale), n, ptrs

    def forward(self, x, h, gamma_post=None, gate=None, gamma_pre=None):
        """(out, y, rstd_post, rstd_pre) for x, h [..., C]; a gain that is None is
        left out, and with it y and rstd_pre (gamma_pre) or rstd_post
        (gamma_post) are None.  gate: [C] or [G, C], G dividing the tokens."""
        cfg, n, gains = self._gains(x, gamma_post, gate, gamma_pre)
        xp = self._rows(x, x.shape, x.device, "x")
        hp = self._rows(h, x.shape, x.device, "h")
        with capi.on_device(x.device):
            out = torch.empty_like(x)
            y = torch.empty_like(x) if gamma_pre is not None else None
            rh = torch.empty(n, dtype=torch.float32, device=x.device) if gamma_post is not None else None
            ro = torch.empty(n, dtype=torch.float32, device=x.device) if gamma_pre is not None else None
            capi.check(capi.lib().mgpt_norm_forward(
                ctypes.byref(cfg), xp, hp, *gains, out.data_ptr(), None if y is None else y.data_ptr(),
                None if rh is None else rh.data_ptr(), None if ro is None else ro.data_ptr(), n,
                capi.stream(x.device)))
        return out, y, rh, ro

    def backward(self, x, h, dout, dy, rstd_post, rstd_pre, gamma_post=None, gate=None, gamma_pre=None):
        """(dx, dh, dgamma_post, dgate, dgamma_pre) for the upstream gradients
        dout of out (None: zero, with gamma_pre) and dy of y (None without
        gamma_pre), from forward's inputs and the rstd it returned; the
        gradient of a gain that is None is None."""
        cfg, n, gains = self._gains(x, gamma_post, gate, gamma_pre)
        ptrs = [self._rows(x, x.shape, x.device, "x"), self._rows(h, x.shape, x.device, "h")]
        for t, need, what in ((rstd_post, gamma_post, "rstd_post"), (rstd_pre, gamma_pre, "rstd_pre")):
            if need is None:
                gains.append(None)
                continue
            if t is None or t.device != x.device or t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
                raise ValueError(f"{what} must be the float32 tensor that forward returned")
            gains.append(t.data_ptr())
        if gamma_pre is not None and dy is None:
            raise ValueError("dy is needed with gamma_pre")
        if gamma_pre is None and dout is None:
            raise ValueError("dout is needed without gamma_pre")
        up = [None if dout is None else self._rows(dout, x.shape, x.device, "dout"),
              None if gamma_pre is None else self._rows(dy, x.shape, x.device, "dy")]
        with capi.on_device(x.device):
            dx, dh = torch.empty_like(x), torch.empty_like(x)
            grads = [None if g is None else torch.empty_like(g) for g in (gamma_post, gate, gamma_pre)]
            need = ctypes.c_size_t()
            capi.check(capi.lib().mgpt_norm_backward_workspace_bytes(ctypes.byref(cfg), n, ctypes.byref(need)))
            ws = torch.empty(need.value, dtype=torch.uint8, device=x.device)
            capi.check(capi.lib().mgpt_norm_backward(
                ctypes.byref(cfg), *ptrs, *gains, *up, dx.data_ptr(), dh.data_ptr(),
                *[None if g is None else g.data_ptr() for g in grads], n, ws.data_ptr() if need.value else None,
                need.value, capi.stream(x.device)))
        return dx, dh, *grads
