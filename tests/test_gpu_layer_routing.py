"""MoELayer with set_routing: the layer run by the caller's rule instead of the engine's router.

x and the router's weights are small whole multiples of powers of two, so that the logits are exact in fp32 and the
choice can be compared as it is.  Outputs go by the layer's own bars (1e-5 relative in fp32, 2e-2 in
bf16, 6e-2 with fp8 weights, as the layer's other tests), gradients by theirs (1e-5 and 2e-2).  With int8 weights a
rounding is max / 127 / sqrt(12) in rms: of rms 1, weights (max 2.7 to 4) 0.6 to 0.9%, x here (max 1, rms 0.65)
0.4%, h (a product of two normal numbers; max 5 to 8) 1.1 to 1.8%.  g and u are each off by x's and the weights',
0.8 to 1%, h by both, 1.2 to 1.4% (silu's slope is up to 1.1), the output by h's, its rounding's and the weights':
1.8 to 2.5%, and bf16's 0.3%: the bar is 3e-2.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_route import reference  # noqa: E402

BAR = {"f32": 1e-5, "bf16": 2e-2, "fp8": 6e-2, "i8": 3e-2}


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


class Case:
    def __init__(self, C, H, E, k, act, weights, seed=1):
        from mgpt_amd.moe import MoELayer
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.C, self.H, self.E, self.k, self.act = C, H, E, k, act
        self.wr = torch.randint(-3, 4, (C, E), generator=gen, device="cuda") / 64.0
        self.br = torch.randint(-2, 3, (E,), generator=gen, device="cuda") / 64.0
        self.W = [r(E, C, H) / C ** 0.5, r(E, C, H) / C ** 0.5, r(E, H, C) / H ** 0.5]
        self.b = [r(E, H) * 0.1, r(E, H) * 0.1, r(E, C) * 0.1]
        self.op = MoELayer(C, H, E, k, act=act, weights=weights)
        params = [self.wr, self.br]
        for e in range(E):
            for W, b in zip(self.W, self.b):
                params += [W[e], b[e]]
        self.op.load_parameters(params)
        self.weights = weights

    def x(self, N, seed=2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randint(-4, 5, (N, self.C), generator=gen, device="cuda") / 4.0
        return x.to(torch.float32 if self.act == "f32" else torch.bfloat16)

    def logits(self, x):
        return (x.double() @ self.wr.double() + self.br.double()).float()

    def experts(self, x, idx, w, W=None, b=None):
        """In 64 bits."""
        W, b = W or [t.double() for t in self.W], b or [t.double() for t in self.b]
        y = torch.zeros(x.shape[0], self.C, dtype=torch.float64, device="cuda")
        for e in range(self.E):
            t, j = (idx == e).nonzero(as_tuple=True)
            if t.numel():
                z = x[t]
                h = torch.nn.functional.silu(z @ W[0][e] + b[0][e]) * (z @ W[1][e] + b[1][e])
                y = y.index_add(0, t, (h @ W[2][e] + b[2][e]) * w[t, j][:, None])
        return y


def rule(E, k, **kw):
    from mgpt_amd.routing import ExpertRouting
    return ExpertRouting(E, k, **kw)


def of(op, logits, bias):
    c = op.config
    return reference(logits, bias, c.top_k, ["softmax", "sigmoid"][c.score], c.groups, c.top_groups, c.group_best,
                     bool(c.renormalise), c.scale)


RULES = [dict(score="sigmoid", groups=4, top_groups=2, scale=2.5), dict(score="softmax"),
         dict(score="softmax", renormalise=False, groups=2, top_groups=1, group_best=1)]


@pytest.mark.parametrize("act,weights", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "fp8"), ("f32", "fp8"), ("bf16", "i8"),
                                         ("f32", "i8")])
@pytest.mark.parametrize("E,k,C", [(8, 2, 64), (16, 4, 128), (64, 8, 256), (96, 4, 100)])
def test_forward(E, k, C, act, weights):
    c = Case(C, 128, E, k, act, weights)
    for kw, biased in zip(RULES, (True, False, True)):
        if E // kw.get("groups", 1) * kw.get("top_groups", 1) < k:
            continue
        op = rule(E, k, **kw)
        bias = torch.randn(E, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 0.05
        bias = bias if biased else None
        c.op.set_routing(op, bias=bias)
        for N in (1, 40, 300, 1500):
            x = c.x(N)
            y = c.op.forward(x)
            r = c.op.routing()
            idx, w, _ = of(op, c.logits(x), bias)
            assert torch.equal(r["topk_idx"].cpu().long(), idx)
            assert (r["topk_p"].double().cpu() - w).abs().max() < 1e-6 * op.config.scale
            assert torch.equal(r["counts"].cpu().long(), torch.bincount(idx.reshape(-1), minlength=E))
            want = c.experts(x.double(), idx.cuda(), w.cuda())
            assert rel(y, want) < BAR[weights]
            # the routing given is the routing made
            assert torch.equal(c.op.forward_routed(x, idx.int().cuda(), r["topk_p"].clone()), y)


def test_block():
    """The fused block: the choice on the normalised rows, which fp32 rounds: rows whose keys are close are left out."""
    for act, weights in (("f32", "f32"), ("bf16", "bf16"), ("bf16", "i8")):
        c = Case(128, 256, 16, 2, act, weights)
        op = rule(16, 2, score="sigmoid")
        c.op.set_routing(op)
        gamma = 1 + 0.1 * torch.randn(128, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
        for N in (50, 700):
            x = c.x(N)
            y = c.op.forward_block(x, gamma)
            n = x.double() * (x.double().square().mean(1, keepdim=True) + 1e-5).rsqrt() * gamma.double()
            l = n @ c.wr.double() + c.br.double()
            idx, w, _ = of(op, l, None)
            top = l.sort(dim=1, descending=True)[0][:, :3]
            sure = (top[:, :-1] - top[:, 1:]).amin(1).cpu() > 1e-4
            r = c.op.routing()
            assert sure.float().mean() > 0.9
            assert torch.equal(r["topk_idx"].cpu().long()[sure], idx[sure])
            want = x.double() + c.experts(n, r["topk_idx"].long(), r["topk_p"].double())
            assert rel(y, want) < BAR[weights]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N", [60, 900])
@pytest.mark.parametrize("kw,biased,balance", [(RULES[0], True, 0.0), (RULES[1], False, 0.3), (RULES[2], True, 0.0),
                                               (dict(score="sigmoid", renormalise=False), False, 0.5)])
def test_training(act, N, kw, biased, balance):
    E, k, C, H = 8, 2, 64, 96
    c = Case(C, H, E, k, act, act)
    op = rule(E, k, **kw)
    bias = (torch.arange(E, device="cuda") % 3 * 0.03) if biased else None
    c.op.set_routing(op, bias=bias, balance=balance)
    x = c.x(N)
    dy = torch.randn(N, C, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(x.dtype)
    c.op.zero_grad()
    y = c.op.forward(x, train=True)
    dx = c.op.backward(dy)
    idx, _, on = of(op, c.logits(x), bias)
    idx, on = idx.cuda(), on.cuda()
    assert torch.equal(c.op.routing()["topk_idx"].long(), idx)
    # the same in 64 bits, differentiated by torch
    xd = x.double().requires_grad_()
    leaves = [t.double().requires_grad_() for t in (c.wr, c.br, *c.W, *c.b)]
    l = xd @ leaves[0] + leaves[1]
    s = torch.softmax(l, 1) if op.config.score == 0 else torch.sigmoid(l)
    sel = s.gather(1, idx) * on
    w = sel * op.config.scale
    if op.config.renormalise:
        w = w / (sel.sum(1, keepdim=True) + 1e-20)
    ref = c.experts(xd, idx, w, leaves[2:5], leaves[5:])
    assert rel(y, ref.detach()) < BAR[act]
    loss = (ref * dy.double()).sum()
    counts = torch.bincount(idx.reshape(-1), minlength=E).double()
    loss = loss + (s * (balance * E * counts / N / N)).sum()
    loss.backward()
    assert rel(dx, xd.grad) < BAR[act]
    got = c.op.get_gradients()
    assert rel(got[0], leaves[0].grad) < BAR[act] and rel(got[1].view(-1), leaves[1].grad) < BAR[act]
    for i in range(3):
        gW = torch.stack([got[2 + 6 * e + 2 * i] for e in range(E)])
        gb = torch.stack([got[3 + 6 * e + 2 * i].view(-1) for e in range(E)])
        assert rel(gW, leaves[2 + i].grad) < BAR[act] and rel(gb, leaves[5 + i].grad) < BAR[act]


def test_training_block_runs():
    c = Case(64, 96, 8, 2, "f32", "f32")
    c.op.set_routing(rule(8, 2, score="sigmoid"))
    x = c.x(100)
    gamma = torch.ones(64, device="cuda")
    out = torch.empty_like(x)
    c.op.zero_grad()
    c.op.forward_block_into(x, gamma, 1e-5, out, train=True)
    r = c.op.routing()
    idx = r["topk_idx"].long().clone()
    dy = torch.randn_like(x)
    dx, dgamma = c.op.backward_block(dy)
    xd, gd = x.double().requires_grad_(), gamma.double().requires_grad_()
    n = xd * (xd.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gd
    s = torch.sigmoid(n @ c.wr.double() + c.br.double()).gather(1, idx)
    ref = xd + c.experts(n, idx, s / (s.sum(1, keepdim=True) + 1e-20))
    (ref * dy.double()).sum().backward()
    assert rel(out, ref.detach()) < 1e-5 and rel(dx, xd.grad) < 1e-5 and rel(dgamma, gd.grad) < 1e-5


def test_back_to_the_engines_router_and_refusals():
    from mgpt_amd import capi
    c = Case(64, 96, 8, 2, "f32", "f32")
    x = c.x(200)
    want = c.op.forward(x).clone()
    c.op.set_routing(rule(8, 2, score="sigmoid"))
    assert not torch.equal(c.op.forward(x), want)
    c.op.forward(x, train=True)
    c.op.set_routing(None)
    with pytest.raises(capi.MoEError):      # the training forward had another rule
        c.op.backward(x)
    assert torch.equal(c.op.forward(x), want)
    c.op.zero_grad()
    c.op.forward(x, train=True)
    c.op.backward(x)
    for bad in (rule(16, 2), rule(8, 3), rule(8, 2, act="bf16"), rule(8, 2, groups=3), rule(8, 2, scale=0.0)):
        with pytest.raises(capi.MoEError):
            c.op.set_routing(bad)
    with pytest.raises(capi.MoEError):
        c.op.set_routing(rule(8, 2), balance=-1.0)
    with pytest.raises(ValueError):
        c.op.set_routing(rule(8, 2), bias=torch.zeros(8))
    assert torch.equal(c.op.forward(x), want)


def test_captured_step_reads_the_bias_as_it_is():
    """A captured forward, the bias updated between replays from the counts."""
    c = Case(64, 96, 16, 4, "bf16", "i8")
    op = rule(16, 4, score="sigmoid")
    bias = torch.zeros(16, device="cuda")
    c.op.set_routing(op, bias=bias)
    for N in (32, 600):
        x = c.x(N)
        c.op.reserve(600)
        c.op.forward(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = c.op.forward(x)
            counts = c.op.routing()["counts"]
            op.balance(bias, counts, 0.05)
        for seed in (4, 5, 6):
            x.copy_(c.x(N, seed))
            before = bias.clone()
            graph.replay()
            torch.cuda.synchronize()
            got, after = y.clone(), bias.clone()
            idx = of(op, c.logits(x), before)[0]
            n = torch.bincount(idx.reshape(-1), minlength=16).double()
            assert torch.equal(after.cpu(), (before.cpu() + 0.05 * torch.sign(n.mean() - n).float()))
            bias.copy_(before)
            assert torch.equal(c.op.forward(x), got)
            bias.copy_(after)
