"""AdamW: one step over all tensors of a model in one launch per 116 of them.

Mirrors the engine's AdamWOptimizer
(/root/reference/src/main/neuralnetwork/optimisers/AdamWOptimiser.h:13-97)
over the C ABI (mgpt_adamw_step).  The moments are fp32 or 8 bits per value;
the parameters are fp32 CUDA tensors, updated in place, e.g. the 2 + 6E
tensors a MoELayer loads, with the gradients of MoELayer.get_gradients().
"""
from __future__ import annotations

import array
import ctypes
import operator

import torch

from . import capi

_GRAD = {torch.float32: capi.DTYPE_F32, torch.bfloat16: capi.DTYPE_BF16}
_dtype = operator.attrgetter("dtype")
_numel, _is_contiguous = torch.Tensor.numel, torch.Tensor.is_contiguous
_get_device, _data_ptr = torch.Tensor.get_device, torch.Tensor.data_ptr


def _addresses(tensors, some):
    """The tensors' addresses, 0 for None, as the C ABI takes them; some: those
    that are not None."""
    ptrs = list(map(_data_ptr, some))
    if len(some) != len(tensors):
        at = iter(ptrs)
        ptrs = [0 if t is None else next(at) for t in tensors]
    return array.array("Q", ptrs)


class AdamW:
    """params: contiguous float32 CUDA tensors of one device, which keep their
    memory.  copies: None, or per parameter a bfloat16 tensor of its size (or
    None) that every step refreshes.  state_bits: 32 or 8.  device_step: keep the
    step's number on the device, so that a step captured into a HIP graph counts
    on when it is replayed; without it a replayed step repeats the number that
    it was captured with.  To go on from a saved run, copy its state into
    `state` and set step_count."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32, copies=None, device_step: bool = False):
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.state_bits = state_bits
        self.device = self.params[0].device
        self.copies = list(copies) if copies is not None else None
        if self.copies is not None and len(self.copies) != len(self.params):
            raise ValueError("copies must have an entry per parameter")
        for i, p in enumerate(self.params):
            self._check(p, torch.float32, p.numel(), f"params[{i}]")
            if self.copies is not None and self.copies[i] is not None:
                self._check(self.copies[i], torch.bfloat16, p.numel(), f"copies[{i}]")
        written = self.params + [c for c in self.copies or [] if c is not None]
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in written if t.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("params and copies must not overlap")
        # aliases: as long as a parameter is still at its address, the memory there is
        # the one that was checked, whatever has been assigned to its .data since
        self._held = [t.detach() for t in written]
        self._at = self._written()
        n = len(self.params)
        self._numels = [p.numel() for p in self.params]
        self._sizes = (ctypes.c_int64 * n)(*self._numels)
        need = ctypes.c_size_t()
        capi.check(capi.lib().mgpt_adamw_state_bytes(n, self._sizes, state_bits, ctypes.byref(need)))
        self.state = torch.zeros(need.value, dtype=torch.uint8, device=self.device)
        self._step_device = (torch.zeros(1, dtype=torch.int32, device=self.device) if device_step else None)
        self._steps = 0   # where the number is not on the device
        blocks = sum((p.numel() + 255) // 256 for p in self.params)
        held = blocks * 256 * state_bits // 8
        kinds = (torch.float32, torch.float32) if state_bits == 32 else (torch.float8_e4m3fn, torch.uint8)
        # views of the state, in its own order (a tensor takes whole blocks of 256)
        self.m = self.state[:held].view(kinds[0])
        self.v = self.state[held:2 * held].view(kinds[1])
        self.m_exp = self.state[2 * held:2 * held + blocks] if state_bits == 8 else None
        self.v_exp = self.state[2 * held + blocks:] if state_bits == 8 else None

    @property
    def step_count(self) -> int:
        """The steps taken; the next is one more.  With device_step it is read
        from the device, which waits for the steps before, and set there."""
        return self._steps if self._step_device is None else int(self._step_device.item())

    @step_count.setter
    def step_count(self, count: int) -> None:
        if self._step_device is None:
            self._steps = count
        else:
            self._step_device.fill_(count)

    def _check(self, t, dtype, numel, what):
        if t.device != self.device or not t.is_cuda:
            raise ValueError(f"{what} must be a CUDA tensor on {self.device}")
        if t.dtype != dtype:
            raise TypeError(f"{what} must be {dtype}")
        if t.numel() != numel or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous with {numel} elements")

    def _written(self):
        """The addresses of the parameters and of their copies (None: no copies)."""
        if self.copies is None:
            return _addresses(self.params, self.params), None
        return (_addresses(self.params, self.params),
                _addresses(self.copies, [c for c in self.copies if c is not None]))

    def step(self, grads, grad_scale: torch.Tensor | None = None) -> None:
        """One step from `grads`: per parameter a contiguous tensor of its size,
        all float32 or all bfloat16, or None (the parameter and its moments
        stay).  grad_scale: float32 device tensor of one element."""
        grads = list(grads)
        n = len(self.params)
        if len(grads) != n:
            raise ValueError(f"expected {n} gradients, got {len(grads)}")
        # (attribute by attribute over all tensors: a model has hundreds, and their
        # checks one by one would take longer than the step)
        some = [g for g in grads if g is not None]
        dtypes = set(map(_dtype, some)) or {torch.float32}
        if len(dtypes) != 1 or not dtypes <= _GRAD.keys():
            raise TypeError("gradients must be all float32 or all bfloat16")
        sizes = self._numels if len(some) == n else [k for k, g in zip(self._numels, grads) if g is not None]
        if list(map(_numel, some)) != sizes or not all(map(_is_contiguous, some)):
            raise ValueError("gradients must be contiguous and have their parameters' sizes")
        if not set(map(_get_device, some)) <= {self.device.index}:
            raise ValueError(f"gradients must be CUDA tensors on {self.device}")
        if self._written() != self._at:
            raise ValueError("a parameter or a copy no longer has the memory it was given with")
        gp, (pp, cp) = _addresses(grads, some), self._at
        scale = None
        if grad_scale is not None:
            self._check(grad_scale, torch.float32, 1, "grad_scale")
            scale = grad_scale.data_ptr()
        cfg = capi.AdamWConfig(self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay,
                               self.state_bits, _GRAD[dtypes.pop()])
        with capi.on_device(self.device):
            number = self._steps + 1
            at = None
            if self._step_device is not None:
                self._step_device.add_(1)
                at = self._step_device.data_ptr()
            status = capi.lib().mgpt_adamw_step(
                ctypes.byref(cfg), n, self._sizes, pp.buffer_info()[0], gp.buffer_info()[0],
                None if cp is None else cp.buffer_info()[0], self.state.data_ptr(), self.state.numel(), number, at,
                scale, capi.stream(self.device))
            if status != capi.MGPT_OK and at is not None:
                self._step_device.sub_(1)   # a refused step is none
            capi.check(status)
        if at is None:
            self._steps = number
