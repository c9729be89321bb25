"""The operators of a training step as a program runs them together: the MoE
layer, the norms around it with gate and residual, the head's loss, their
backwards and AdamW over every parameter, with the layer re-loaded after each
step.  Against 64 bits: the gradients of norm and loss by automatic
differentiation of the plain formulas, from the layer's own output; each
step's update by AdamW's formula; the layer after the steps against a new one
loaded with the same parameters.  A captured loss-norm-AdamW step replays to the
eager one's bits."""
import numpy as np
import pytest

from mgpt_amd import workload as wl

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


def plain(x, h, post, gate, pre, W, b, t, s):
    """Mean loss in the inputs' precision (64 bits here)."""
    n = h * (h.square().mean(1, keepdim=True) + EPS).rsqrt()
    o = s * x + gate * (n * post)
    y = o * (o.square().mean(1, keepdim=True) + EPS).rsqrt() * pre
    z = y @ W.t() + b
    has = (t >= 0) & (t < W.shape[0])
    return torch.nn.functional.cross_entropy(z[has], t[has].long())


@pytest.mark.parametrize("act,bits", [("f32", 32), ("f32", 8), ("bf16", 32)])
def test_steps_of_a_small_model(act, bits):
    from mgpt_amd.loss import LMLoss
    from mgpt_amd.moe import MoELayer
    from mgpt_amd.norm import ResidualNorm
    from mgpt_amd.optim import AdamW
    N, C, E, k, H, V, s = 200, 64, 4, 2, 96, 333, 0.5
    cfg = wl.MoEConfig("step", N, C, E, k, H, act, act, "normal")
    inp = wl.make_inputs(cfg, seed=3, bias_std=0.05)
    dt = torch.float32 if act == "f32" else torch.bfloat16
    gen = torch.Generator().manual_seed(1)
    # fp32 parameters; the layer and the head run on copies of them in dt
    params = [torch.from_numpy(np.ascontiguousarray(p, np.float32)).cuda() for p in inp.params(raw=True)]
    W = (torch.randn(V, C, generator=gen) * 0.1).cuda()
    b = torch.zeros(V, device="cuda")
    post, pre = torch.ones(C, device="cuda"), torch.ones(C, device="cuda")
    gate = torch.full((C,), 0.3, device="cuda")
    x = torch.from_numpy(inp.x).cuda().to(dt)
    t = torch.randint(0, V, (N,), generator=gen, dtype=torch.int32).cuda()
    t[::9] = -1
    Wc = W.to(dt) if act == "bf16" else W
    copies = [None] * len(params) + ([Wc] if act == "bf16" else [None]) + [None] * 4
    every = params + [W, b, post, gate, pre]
    opt = AdamW(every, lr=1e-2, state_bits=bits, copies=copies)
    layer = MoELayer(C, H, E, k, act=act)
    norm, head = ResidualNorm(C, act=act, eps=EPS, residual_scale=s), LMLoss(C, V, act=act)
    losses = []
    for step in range(4):
        layer.load_parameters(params)
        layer.zero_grad()
        h = layer.forward(x, train=True)
        out, y, rh, ro = norm.forward(x, h, gamma_post=post, gate=gate, gamma_pre=pre)
        loss, lse, mean = head.forward(y, Wc, t, bias=b)
        dy, dW, db = head.backward(y, Wc, t, lse, bias=b)
        dx, dh, dpost, dgate, dpre = norm.backward(x, h, None, dy, rh, ro, gamma_post=post, gate=gate, gamma_pre=pre)
        layer.backward(dh)
        grads = layer.get_gradients() + [dW.float(), db, dpost, dgate, dpre]
        # in 64 bits from the layer's output
        leaves = [v.double().detach().requires_grad_() for v in (x, h, post, gate, pre, Wc, b)]
        ref = plain(*leaves, t, s)
        ref.backward()
        losses.append(float(mean[0]))
        # every operator's own error is tested elsewhere; in bf16 y, dy and the outputs
        # carry half a step (2^-8) each, through at most 4 such tensors in a row
        tol = 1e-5 if act == "f32" else 4 * 2.0 ** -8
        assert abs(losses[-1] - ref.item()) <= tol * ref.item()
        for name, got, leaf in zip(("dx", "dh", "dpost", "dgate", "dpre", "dW", "db"),
                                   (dx, dh, dpost, dgate, dpre, dW, db), leaves):
            want = leaf.grad.reshape(got.shape)
            err = float((got.double() - want).norm() / want.norm())
            assert err <= tol, (step, name, err)
        before = [p.clone() for p in every]
        if bits == 32:
            sl, at = [], 0
            for p in every:
                sl.append(slice(at, at + p.numel()))
                at += (p.numel() + 255) // 256 * 256
            m0, v0 = opt.m.double(), opt.v.double()
        opt.step([g.contiguous() for g in grads])
        if bits == 32:
            b1, b2, lr, eps, wd = (float(np.float32(q)) for q in (0.9, 0.999, 1e-2, 1e-8, 0.01))
            for p, q, g, r in zip(every, before, grads, sl):
                g = g.double().reshape(-1)
                m = b1 * m0[r] + (1 - b1) * g
                v = b2 * v0[r] + (1 - b2) * g * g
                want = q.double().reshape(-1) * (1 - lr * wd) - lr * (m / (1 - b1 ** (step + 1))) / (
                    (v / (1 - b2 ** (step + 1))).sqrt() + eps)
                # an update is at most 10 lr; 16 roundings of it, 3 of the parameter
                err = (p.double().reshape(-1) - want).abs()
                assert (err <= 3 * 2.0 ** -24 * (want.abs() + q.double().reshape(-1).abs()) + 160 * 2.0 ** -24 * lr).all()
        if act == "bf16":
            assert torch.equal(Wc, W.bfloat16())
    assert all(np.isfinite(losses))
    # the layer computes with the parameters that the last step left
    layer.load_parameters(params)
    fresh = MoELayer(C, H, E, k, act=act)
    fresh.load_parameters([p.cpu().numpy() for p in params])
    assert torch.equal(layer.forward(x), fresh.forward(x))


def test_captured_step():
    """Norm, loss, their backwards and AdamW captured once and replayed, with
    eager steps on the same shapes between the replays."""
    from mgpt_amd.loss import LMLoss
    from mgpt_amd.norm import ResidualNorm
    from mgpt_amd.optim import AdamW
    N, C, V = 300, 128, 1000
    gen = torch.Generator().manual_seed(2)

    def model(device_step):
        g = torch.Generator().manual_seed(7)
        p = {"W": (torch.randn(V, C, generator=g) * 0.1).cuda(), "post": torch.ones(C, device="cuda"),
             "pre": torch.ones(C, device="cuda"), "gate": torch.ones(C, device="cuda")}
        opt = AdamW(list(p.values()), lr=1e-2, state_bits=8, device_step=device_step)
        return p, opt

    norm, head = ResidualNorm(C, act="f32", eps=EPS), LMLoss(C, V, act="f32")
    x, h = torch.randn(N, C, generator=gen).cuda(), torch.randn(N, C, generator=gen).cuda()
    t = torch.randint(-1, V, (N,), generator=gen, dtype=torch.int32).cuda()

    def step(p, opt, x, h):
        kw = dict(gamma_post=p["post"], gate=p["gate"], gamma_pre=p["pre"])
        out, y, rh, ro = norm.forward(x, h, **kw)
        loss, lse, mean = head.forward(y, p["W"], t)
        dy, dW, _ = head.backward(y, p["W"], t, lse)
        dx, dh, dpost, dgate, dpre = norm.backward(x, h, None, dy, rh, ro, **kw)
        opt.step([dW, dpost, dpre, dgate])
        return mean

    pe, oe = model(False)
    pc, oc = model(True)
    xs, hs = x.clone(), h.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mean = step(pc, oc, xs, hs)
    for i in range(4):
        xi, hi = x * (1 + i), h.roll(i, 0).contiguous()
        want = step(pe, oe, xi, hi)
        xs.copy_(xi)
        hs.copy_(hi)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mean, want), i
        for k in pe:
            assert torch.equal(pe[k], pc[k]), (i, k)
        assert torch.equal(oe.state, oc.state), i
