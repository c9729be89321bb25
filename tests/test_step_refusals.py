"""What the operators of the training step refuse, before anything runs: the C
ABI with bad sizes, types, null pointers and small workspaces (no address is
read), and the Python classes with tensors that are not on the GPU."""
import ctypes

import pytest

from mgpt_amd import capi

torch = pytest.importorskip("torch")

INV, UNS, SMALL = capi.MGPT_ERR_INVALID_ARGUMENT, capi.MGPT_ERR_UNSUPPORTED, capi.MGPT_ERR_WORKSPACE_TOO_SMALL
P = ctypes.c_void_p(1 << 20)     # an aligned address that is never read
ODD = ctypes.c_void_p((1 << 20) + 2)


def refused(status, want):
    assert status == want and capi.lib().mgpt_moe_last_error().decode()


# ------------------------------------------------------------------- AdamW
def adamw(cfg=None, sizes=(5, 300), params=None, grads=None, copies=None, state=P, state_bytes=1 << 20, step=1, n=None,
          step_device=None):
    k = len(sizes)
    cfg = cfg or capi.AdamWConfig(1e-3, 0.9, 0.999, 1e-8, 0.01, 32, capi.DTYPE_F32)
    array = ctypes.c_void_p * k
    pp = array(*[P.value] * k) if params is None else params
    gp = array(*[P.value] * k) if grads is None else grads
    return capi.lib().mgpt_adamw_step(ctypes.byref(cfg) if cfg != "null" else None, k if n is None else n,
                                      (ctypes.c_int64 * k)(*sizes), pp, gp, copies, state, state_bytes, step,
                                      step_device, None, None)


def config(**kw):
    c = capi.AdamWConfig(1e-3, 0.9, 0.999, 1e-8, 0.01, 32, capi.DTYPE_F32)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw", [dict(beta1=1.0), dict(beta2=-0.1), dict(beta2=float("nan")), dict(eps=-1.0),
                                dict(eps=float("nan")), dict(lr=float("inf")), dict(weight_decay=float("nan"))])
def test_adamw_refuses_hyperparameters(kw):
    refused(adamw(config(**kw)), INV)


def test_adamw_refuses_arguments():
    refused(adamw(config(state_bits=16)), UNS)
    refused(adamw(config(grad_dtype=capi.DTYPE_FP8_E4M3)), UNS)
    refused(adamw("null"), INV)
    refused(adamw(n=-1), INV)
    refused(adamw(sizes=(5, -1)), INV)
    refused(adamw(sizes=((1 << 34) + 1,)), INV)
    refused(adamw(step=0), INV)
    refused(adamw(state=None), INV)
    refused(adamw(state=ODD), INV)
    refused(adamw(state_bytes=2 * 256 * 3 * 4 - 1), SMALL)
    refused(adamw(params=(ctypes.c_void_p * 2)(P.value, None)), INV)
    refused(adamw(params=(ctypes.c_void_p * 2)(P.value, ODD.value)), INV)
    refused(adamw(grads=(ctypes.c_void_p * 2)(P.value, ODD.value)), INV)
    refused(adamw(copies=(ctypes.c_void_p * 2)(P.value, P.value + 1)), INV)


def test_adamw_state_bytes():
    need = ctypes.c_size_t()
    sizes = (ctypes.c_int64 * 3)(0, 1, 257)
    call = capi.lib().mgpt_adamw_state_bytes
    assert call(3, sizes, 32, ctypes.byref(need)) == 0 and need.value == 3 * 256 * 8
    assert call(3, sizes, 8, ctypes.byref(need)) == 0 and need.value == 3 * (256 * 2 + 2)
    assert call(0, None, 8, ctypes.byref(need)) == 0 and need.value == 0
    refused(call(3, None, 32, ctypes.byref(need)), INV)
    refused(call(3, sizes, 4, ctypes.byref(need)), UNS)
    refused(call(3, sizes, 32, None), INV)
    # nothing to do is no error and touches nothing
    assert adamw(sizes=(0, 0), state=None) == 0


# ------------------------------------------------------------------- norms
def norm_forward(cfg, x=P, h=P, post=P, gate=P, pre=P, out=P, y=P, rh=P, ro=P, n=12):
    return capi.lib().mgpt_norm_forward(ctypes.byref(cfg) if cfg else None, x, h, post, gate, pre, out, y, rh, ro, n,
                                        None)


def norm_backward(cfg, x=P, h=P, post=P, gate=P, pre=P, rh=P, ro=P, dout=P, dy=P, dx=P, dh=P, dpost=P, dgate=P, dpre=P,
                  n=12, ws=P, nbytes=1 << 30):
    return capi.lib().mgpt_norm_backward(ctypes.byref(cfg) if cfg else None, x, h, post, gate, pre, rh, ro, dout, dy,
                                         dx, dh, dpost, dgate, dpre, n, ws, nbytes, None)


@pytest.mark.parametrize("fields,want", [
    ((0, 0, 1, 1e-5, 1.0), INV), ((16385, 0, 1, 1e-5, 1.0), UNS), ((64, 2, 1, 1e-5, 1.0), UNS),
    ((64, 0, 0, 1e-5, 1.0), INV), ((64, 0, 5, 1e-5, 1.0), INV), ((64, 0, 1, -1.0, 1.0), INV),
    ((64, 0, 1, float("nan"), 1.0), INV), ((64, 0, 1, 1e-5, float("inf")), INV)])
def test_norm_refuses_configs(fields, want):
    cfg = capi.NormConfig(*fields)
    refused(norm_forward(cfg), want)
    refused(norm_backward(cfg), want)


def test_norm_refuses_arguments():
    cfg = capi.NormConfig(64, 0, 4, 1e-5, 1.0)
    refused(norm_forward(None), INV)
    refused(norm_forward(cfg, n=-4), INV)
    refused(norm_forward(cfg, n=(1 << 30) + 4), UNS)
    for k in ("x", "h", "out", "y", "rh", "ro"):
        refused(norm_forward(cfg, **{k: None}), INV)
    for k in ("x", "h", "dy", "dx", "dh", "rh", "ro", "ws"):
        refused(norm_backward(cfg, **{k: None}), INV)
    for k in ("post", "gate", "pre"):   # their gradients are asked for
        refused(norm_backward(cfg, **{k: None}), INV)
    refused(norm_backward(cfg, pre=None, dpre=None, dout=None), INV)
    refused(norm_backward(cfg, ws=ctypes.c_void_p((1 << 20) + 64)), INV)
    need = ctypes.c_size_t()
    assert capi.lib().mgpt_norm_backward_workspace_bytes(ctypes.byref(cfg), 12, ctypes.byref(need)) == 0
    refused(norm_backward(cfg, nbytes=64), SMALL)
    refused(capi.lib().mgpt_norm_backward_workspace_bytes(ctypes.byref(cfg), 12, None), INV)
    assert norm_forward(cfg, n=0, x=None) == 0


# -------------------------------------------------------------------- loss
def loss_forward(cfg, x=P, W=P, b=P, t=P, loss=P, lse=P, mean=P, n=10, ws=P, nbytes=1 << 40):
    return capi.lib().mgpt_lm_loss_forward(ctypes.byref(cfg) if cfg else None, x, W, b, t, loss, lse, mean, n, ws,
                                           nbytes, None)


def loss_backward(cfg, x=P, W=P, b=P, t=P, lse=P, dloss=None, dmean=None, dx=P, dW=P, db=P, n=10, ws=P,
                  nbytes=1 << 40):
    return capi.lib().mgpt_lm_loss_backward(ctypes.byref(cfg) if cfg else None, x, W, b, t, lse, dloss, dmean, dx, dW,
                                            db, n, ws, nbytes, None)


@pytest.mark.parametrize("fields,want", [((0, 8, 0), INV), ((8, 0, 0), INV), ((8, 8, 2), UNS), ((8, 8, -1), UNS),
                                         (((1 << 20) + 1, 8, 0), UNS), ((8, (1 << 24) + 1, 0), UNS)])
def test_loss_refuses_configs(fields, want):
    cfg = capi.LMLossConfig(*fields)
    refused(loss_forward(cfg), want)
    refused(loss_backward(cfg), want)
    need = ctypes.c_size_t()
    refused(capi.lib().mgpt_lm_loss_workspace_bytes(ctypes.byref(cfg), 4, ctypes.byref(need)), want)


@pytest.mark.parametrize("dtype", [capi.DTYPE_F32, capi.DTYPE_BF16])
def test_loss_refuses_arguments(dtype):
    cfg = capi.LMLossConfig(64, 100, dtype)
    refused(loss_forward(None), INV)
    refused(loss_backward(None), INV)
    refused(loss_forward(cfg, n=-1), INV)
    refused(loss_forward(cfg, n=(1 << 21) + 1), UNS)
    for k in ("x", "W", "t", "loss", "lse", "ws"):
        refused(loss_forward(cfg, **{k: None}), INV)
    for k in ("x", "W", "t", "lse", "ws"):
        refused(loss_backward(cfg, **{k: None}), INV)
    refused(loss_backward(cfg, dloss=P, dmean=P), INV)
    refused(loss_forward(cfg, ws=ctypes.c_void_p((1 << 20) + 16)), INV)
    for query, call in ((capi.lib().mgpt_lm_loss_workspace_bytes, loss_forward),
                        (capi.lib().mgpt_lm_loss_backward_workspace_bytes, loss_backward)):
        need = ctypes.c_size_t()
        assert query(ctypes.byref(cfg), 10, ctypes.byref(need)) == 0 and need.value > 0
        refused(call(cfg, nbytes=256), SMALL)
        refused(query(ctypes.byref(cfg), 10, None), INV)
    # no gradient is wanted: nothing to do
    assert loss_backward(cfg, dx=None, dW=None, db=None) == 0


def test_the_workspace_does_not_grow_past_its_pieces():
    """Backward workspaces hold a piece of the vocabulary, not all of it."""
    need = ctypes.c_size_t()
    for V in (1 << 17, 1 << 20):
        cfg = capi.LMLossConfig(1024, V, capi.DTYPE_BF16)
        assert capi.lib().mgpt_lm_loss_backward_workspace_bytes(ctypes.byref(cfg), 16384, ctypes.byref(need)) == 0
        assert need.value < 3 << 30


# ------------------------------------------------------------------ Python
def test_python_classes_refuse_cpu_tensors():
    from mgpt_amd.loss import LMLoss
    from mgpt_amd.norm import ResidualNorm
    from mgpt_amd.optim import AdamW
    with pytest.raises(ValueError):
        AdamW([torch.zeros(4)])
    with pytest.raises(ValueError):
        AdamW([])
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        ResidualNorm(8, act="f32").forward(x, x)
    with pytest.raises(ValueError):
        ResidualNorm(9, act="f32").forward(x, x)
    with pytest.raises(ValueError):
        LMLoss(8, 3, act="f32").forward(x, torch.zeros(3, 8), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(KeyError):
        LMLoss(8, 3, act="f16")
