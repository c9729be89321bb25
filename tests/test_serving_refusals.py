"""What routing, the integer linear layer and sampling refuse, before anything runs: the C ABI with bad sizes, types, null
pointers and small workspaces (no address is read), and the Python classes with tensors that are not on the GPU."""
import ctypes

import pytest

from mgpt_amd import capi

torch = pytest.importorskip("torch")

INV, UNS, SMALL = capi.MGPT_ERR_INVALID_ARGUMENT, capi.MGPT_ERR_UNSUPPORTED, capi.MGPT_ERR_WORKSPACE_TOO_SMALL
P = ctypes.c_void_p(1 << 20)     # an aligned address that is never read
ODD = ctypes.c_void_p((1 << 20) + 2)
F32, BF16, FP8 = capi.DTYPE_F32, capi.DTYPE_BF16, capi.DTYPE_FP8_E4M3


def refused(status, want):
    assert status == want and capi.lib().mgpt_moe_last_error().decode()


def with_(cfg, **kw):
    for k, v in kw.items():
        setattr(cfg, k, v)
    return cfg


def ref(cfg):
    return None if cfg is None else ctypes.byref(cfg)


# ----------------------------------------------------------------- routing
def route(**kw):
    return with_(capi.RouteConfig(64, 8, capi.SCORE_SIGMOID, 8, 4, 2, 1, 2.5, F32), **kw)


def route_forward(cfg, n=5, logits=P, idx=P, weights=P):
    return capi.lib().mgpt_route_forward(ref(cfg), logits, None, idx, weights, None, n, None)


def route_backward(cfg, n=5, logits=P, idx=P, weights=P, dweights=P, dlogits=P):
    return capi.lib().mgpt_route_backward(ref(cfg), logits, idx, weights, dweights, None, dlogits, n, None)


BAD_ROUTES = [(dict(num_experts=0), INV), (dict(num_experts=513, groups=1, top_groups=1), UNS), (dict(top_k=0), INV),
              (dict(top_k=9), UNS), (dict(num_experts=4, groups=1, top_groups=1), INV), (dict(score=2), INV),
              (dict(groups=0), INV), (dict(groups=7), INV), (dict(top_groups=0), INV), (dict(top_groups=9), INV),
              (dict(num_experts=256, groups=128, top_groups=4), UNS), (dict(group_best=0), INV), (dict(group_best=3), INV),
              (dict(scale=0.0), INV), (dict(scale=float("nan")), INV), (dict(scale=float("inf")), INV),
              (dict(dtype=FP8), UNS), (dict(dtype=capi.DTYPE_I8), UNS)]


@pytest.mark.parametrize("kw,want", BAD_ROUTES)
def test_route_refuses_configs(kw, want):
    refused(route_forward(route(**kw)), want)
    refused(route_backward(route(**kw)), want)
    refused(route_forward(route(**kw), n=0), want)


def test_route_refuses_arguments():
    for f, names in ((route_forward, ("logits", "idx", "weights")),
                     (route_backward, ("logits", "idx", "weights", "dweights", "dlogits"))):
        refused(f(None), INV)
        refused(f(route(), n=-1), INV)
        refused(f(route(), n=(1 << 28) + 1), UNS)
        for name in names:
            refused(f(route(), **{name: None}), INV)
        assert f(route(), n=0, **{name: None for name in names}) == 0
    balance = capi.lib().mgpt_route_balance
    refused(balance(0, P, 0.1, P, None), INV)
    refused(balance(513, P, 0.1, P, None), UNS)
    refused(balance(8, P, float("nan"), P, None), INV)
    refused(balance(8, None, 0.1, P, None), INV)
    refused(balance(8, P, 0.1, None, None), INV)


def test_layer_refuses_null_handles():
    refused(capi.lib().mgpt_moe_set_routing(None, ctypes.byref(route()), None, 0.0), INV)
    refused(capi.lib().mgpt_moe_forward_routed(None, P, P, P, P, 5, P, 1 << 20, None), INV)


def test_routing_refuses_tensors():
    from mgpt_amd.routing import ExpertRouting
    r = ExpertRouting(64, 8)
    l, w = torch.zeros(3, 64), torch.zeros(3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        r.forward(l)
    with pytest.raises(ValueError, match="columns"):
        r.forward(torch.zeros(3, 63))
    with pytest.raises(ValueError, match="CUDA"):
        r.backward(l, torch.zeros(3, 8, dtype=torch.int32), w, w)
    with pytest.raises(ValueError, match="CUDA"):
        r.balance(torch.zeros(64), torch.zeros(64, dtype=torch.int32), 0.1)
    with pytest.raises(KeyError):
        ExpertRouting(64, 8, score="tanh")
    with pytest.raises(KeyError):
        ExpertRouting(64, 8, act="f16")


# ------------------------------------------------------------------ linear
def linear(**kw):
    return with_(capi.I8Config(96, 40, BF16), **kw)


def need(cfg, n):
    out = ctypes.c_size_t()
    assert capi.lib().mgpt_i8_linear_workspace_bytes(ref(cfg), n, ctypes.byref(out)) == 0
    return out.value


def linear_forward(cfg, x=P, packed=P, scales=P, y=P, n=5, ws=P, size=1 << 30):
    return capi.lib().mgpt_i8_linear_forward(ref(cfg), x, packed, scales, None, y, n, ws, size, None)


@pytest.mark.parametrize("kw,want", [(dict(in_features=0), INV), (dict(out_features=0), INV), (dict(in_features=-3), INV),
                                     (dict(in_features=(1 << 17) + 1), UNS), (dict(out_features=(1 << 24) + 1), UNS),
                                     (dict(dtype=FP8), UNS), (dict(dtype=9), UNS)])
def test_linear_refuses_configs(kw, want):
    size = ctypes.c_size_t()
    L = capi.lib()
    refused(linear_forward(linear(**kw)), want)
    refused(L.mgpt_i8_weight_bytes(ref(linear(**kw)), ctypes.byref(size)), want)
    refused(L.mgpt_i8_linear_workspace_bytes(ref(linear(**kw)), 5, ctypes.byref(size)), want)
    refused(L.mgpt_i8_pack_weight(ref(linear(**kw)), P, F32, P, P, None), want)
    refused(L.mgpt_i8_pack_quantized(ref(linear(**kw)), P, P, None), want)


def test_linear_refuses_arguments():
    L = capi.lib()
    size = ctypes.c_size_t()
    for f in (lambda c: linear_forward(c), lambda c: L.mgpt_i8_weight_bytes(ref(c), ctypes.byref(size)),
              lambda c: L.mgpt_i8_pack_weight(ref(c), P, F32, P, P, None), lambda c: L.mgpt_i8_pack_quantized(ref(c), P, P, None)):
        refused(f(None), INV)
    refused(L.mgpt_i8_weight_bytes(ref(linear()), None), INV)
    refused(L.mgpt_i8_linear_workspace_bytes(ref(linear()), 5, None), INV)
    refused(L.mgpt_i8_pack_weight(ref(linear()), None, F32, P, P, None), INV)
    refused(L.mgpt_i8_pack_weight(ref(linear()), P, F32, None, P, None), INV)
    refused(L.mgpt_i8_pack_weight(ref(linear()), P, F32, P, None, None), INV)
    refused(L.mgpt_i8_pack_weight(ref(linear()), P, F32, ODD, P, None), INV)
    refused(L.mgpt_i8_pack_weight(ref(linear()), P, FP8, P, P, None), UNS)
    refused(L.mgpt_i8_pack_quantized(ref(linear()), None, P, None), INV)
    refused(L.mgpt_i8_pack_quantized(ref(linear()), P, None, None), INV)
    refused(L.mgpt_i8_pack_quantized(ref(linear()), P, ODD, None), INV)
    for name in ("x", "packed", "scales", "y", "ws"):
        refused(linear_forward(linear(), **{name: None}), INV)
    refused(linear_forward(linear(), ws=ODD), INV)
    refused(linear_forward(linear(), packed=ODD), INV)
    refused(linear_forward(linear(), n=-1), INV)
    refused(linear_forward(linear(), n=(1 << 21) + 1), UNS)
    refused(linear_forward(linear(), size=need(linear(), 5) - 1), SMALL)
    assert linear_forward(linear(), x=None, y=None, n=0, ws=None, size=0) == 0


def test_linear_refuses_tensors():
    from mgpt_amd.linear8 import I8Linear
    layer = I8Linear(96, 40)
    with pytest.raises(RuntimeError, match="no weight"):
        layer.forward(torch.zeros(2, 96, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        layer.load(torch.zeros(40, 96))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        layer.load(torch.zeros(40, 96, dtype=torch.float64))
    with pytest.raises(ValueError, match="CUDA"):
        layer.load_quantized(torch.zeros(40, 96, dtype=torch.int8), torch.ones(40))
    with pytest.raises(TypeError, match="int8"):
        layer.load_quantized(torch.zeros(40, 96), torch.ones(40))


# ---------------------------------------------------------------- sampling
def sample(**kw):
    return with_(capi.SampleConfig(50000, F32, 1.0, 0, 1.0, 0.0), **kw)


def run_sample(cfg, logits=P, u=P, token=P, n=5, ws=P, size=1 << 30):
    return capi.lib().mgpt_sample(ref(cfg), logits, u, None, None, None, None, token, None, n, ws, size, None)


@pytest.mark.parametrize("kw,want", [(dict(vocab_size=0), INV), (dict(vocab_size=(1 << 20) + 1), UNS), (dict(dtype=FP8), UNS),
                                     (dict(temperature=-1.0), INV), (dict(temperature=float("nan")), INV),
                                     (dict(top_p=-0.1), INV), (dict(top_p=float("nan")), INV), (dict(min_p=-0.1), INV),
                                     (dict(min_p=float("nan")), INV)])
def test_sample_refuses_configs(kw, want):
    refused(run_sample(sample(**kw)), want)
    refused(run_sample(sample(**kw), n=0), want)


def test_sample_refuses_arguments():
    refused(run_sample(None), INV)
    refused(run_sample(sample(), n=-1), INV)
    refused(run_sample(sample(), n=(1 << 24) + 1), UNS)
    for name in ("logits", "u", "token", "ws"):
        refused(run_sample(sample(), **{name: None}), INV)
    refused(run_sample(sample(), ws=ODD), INV)
    size = ctypes.c_size_t()
    bytes_ = capi.lib().mgpt_sample_workspace_bytes
    refused(bytes_(None, 5, ctypes.byref(size)), INV)
    refused(bytes_(ref(sample()), 5, None), INV)
    refused(bytes_(ref(sample()), -1, ctypes.byref(size)), INV)
    assert bytes_(ref(sample()), 5, ctypes.byref(size)) == 0 and size.value > 0
    refused(run_sample(sample(), size=size.value - 1), SMALL)
    # short rows need none, and no rows nothing at all
    assert bytes_(ref(sample(vocab_size=8192)), 5, ctypes.byref(size)) == 0 and size.value == 0
    assert run_sample(sample(), logits=None, u=None, token=None, n=0, ws=None, size=0) == 0


def test_sampler_refuses_tensors():
    from mgpt_amd.sampling import Sampler
    op = Sampler(100)
    with pytest.raises(ValueError, match="CUDA"):
        op.forward(torch.zeros(2, 100), torch.zeros(2))
    with pytest.raises(ValueError, match="columns"):
        op.forward(torch.zeros(2, 99), torch.zeros(2))
    with pytest.raises(KeyError):
        Sampler(100, act="f16")
