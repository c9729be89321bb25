"""The operators of serving together, as a decode step uses them: routing by the caller's rule inside an MoE block with
experts in 8-bit integers, the head in 8-bit integers, sampling.  The step runs eagerly and from a captured graph,
tokens fed back; every part is held to its own definition on what the parts before it gave."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_i8_linear import quantised  # noqa: E402
from test_gpu_layer_routing import Case, rel, rule  # noqa: E402
from test_gpu_sample import check as check_sample  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


class Model:
    def __init__(self, C=256, H=352, E=16, k=4, V=20011, seed=3):
        from mgpt_amd.linear8 import I8Linear
        from mgpt_amd.sampling import Sampler
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.case = Case(C, H, E, k, "bf16", "i8", seed)
        self.layer = self.case.op
        self.bias = r(E) * 0.05
        self.layer.set_routing(rule(E, k, score="sigmoid", groups=4, top_groups=2, scale=1.5), bias=self.bias)
        self.embedding = r(V, C).bfloat16()
        self.gamma = torch.ones(C, device="cuda")
        self.W, self.b = r(V, C) / C ** 0.5, r(V) * 0.1
        self.head = I8Linear(C, V)
        self.head.load(self.W, self.b)
        self.sampler = Sampler(V, act="bf16")
        self.V = V

    def step(self, token, u, T, k):
        x = self.layer.forward_block(self.embedding[token.long()], self.gamma)
        logits = self.head.forward(x)
        token, logp = self.sampler.forward(logits, u, temperature=T, top_k=k, top_p=0.95, min_p=0.01)
        return x, logits, token, logp


@pytest.mark.parametrize("B", [1, 7, 40])
def test_decode(B):
    m = Model()
    gen = torch.Generator(device="cuda").manual_seed(B)
    T = 0.5 + torch.rand(B, generator=gen, device="cuda")
    k = torch.randint(0, 80, (B,), generator=gen, device="cuda", dtype=torch.int32)
    start = torch.randint(0, m.V, (B,), generator=gen, device="cuda", dtype=torch.int32)
    us = torch.rand(6, B, generator=gen, device="cuda")
    m.layer.reserve(64, device="cuda")
    eager, token = [], start
    for u in us:
        eager.append(m.step(token, u, T, k))
        token = eager[-1][2]

    # each part by its definition, on what the device gave before it
    x, logits, _, _ = eager[0]
    q, sx = quantised(x)
    w, sw = quantised(m.W)
    want = (q @ w.t()) * sx[:, None] * sw + m.b.double()
    mag = (q.abs() @ w.abs().t()) * sx[:, None] * sw + m.b.double().abs()
    assert ((logits.double() - want).abs() <= 2.0 ** -8 * want.abs() + 6 * 2.0 ** -24 * mag).all()
    check_sample(logits, us[0], T, k, 0.95, 0.01)

    # captured whole, tokens fed back inside the buffers, eager steps on other tokens in between
    token, u = start.clone(), us[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(token, u, T, k)
    for i, want in enumerate(eager):
        u.copy_(us[i])
        graph.replay()
        for got, w in zip(out, want):
            assert torch.equal(got, w)
        token.copy_(out[2])
        torch.cuda.synchronize()
        m.step(torch.flip(token, [0]), us[i], T, k)
    assert len({int(t) for t in torch.cat([e[2] for e in eager])}) > 1


def test_a_rule_set_or_its_routing_given():
    """The layer with the rule set, and the rule's own outputs given to the layer: the same bits."""
    from mgpt_amd.routing import ExpertRouting
    for weights, act in (("i8", "bf16"), ("i8", "f32"), ("bf16", "bf16"), ("f32", "f32")):
        c = Case(192, 160, 32, 4, act, weights)
        r = ExpertRouting(32, 4, score="sigmoid", groups=4, top_groups=2)
        bias = torch.linspace(-0.1, 0.1, 32, device="cuda")
        for N in (1, 33, 700):
            x = c.x(N)
            counts = torch.zeros(32, dtype=torch.int32, device="cuda")
            idx, w = r.forward(c.logits(x), bias, counts)
            given = c.op.forward_routed(x, idx, w)
            c.op.set_routing(r, bias)
            ruled = c.op.forward(x)
            assert torch.equal(c.op.routing()["topk_idx"], idx) and torch.equal(c.op.routing()["counts"], counts)
            c.op.set_routing(None)
            assert torch.equal(given, ruled)
            assert rel(given, c.experts(x.double(), idx, w.double())) < {"i8": 3e-2, "bf16": 2e-2, "f32": 1e-5}[weights]


def test_training_steps_even_the_load():
    """Routing, its gradient by hand into the router's weights, and the bias that evens the load: against the same
    steps in 64 bits, the choice taken from the device."""
    from mgpt_amd.routing import ExpertRouting
    gen = torch.Generator(device="cuda").manual_seed(9)
    N, C, E, k = 2048, 64, 16, 2
    r = ExpertRouting(E, k, renormalise=True)
    x = torch.randn(N, C, generator=gen, device="cuda")
    wr = torch.randn(C, E, generator=gen, device="cuda") * 0.1 + torch.linspace(-0.2, 0.2, E, device="cuda")
    target = torch.rand(N, k, generator=gen, device="cuda")
    bias = torch.zeros(E, device="cuda")
    first = None
    for step in range(40):
        logits = x @ wr
        counts = torch.zeros(E, dtype=torch.int32, device="cuda")
        idx, w = r.forward(logits, bias, counts)
        dw = (w - target) / N
        grad = r.backward(logits, idx, w, dw)
        ld = logits.double().requires_grad_()
        p = torch.softmax(ld, 1).gather(1, idx.long())
        p = p / p.sum(1, keepdim=True)
        (p * dw.double()).sum().backward()
        assert rel(grad, ld.grad) < 1e-5
        wr -= 0.5 * (x.t() @ grad)
        r.balance(bias, counts, 0.02)
        spread = (counts.max() - counts.min()).item()
        first = spread if first is None else first
    assert int(counts.sum()) == N * k and spread < first


def test_a_row_without_a_batch_and_no_rows():
    """Tensors of one dimension, and none: the values of a batch of one, and empty outputs."""
    from mgpt_amd.linear8 import I8Linear
    from mgpt_amd.routing import ExpertRouting
    from mgpt_amd.sampling import Sampler
    gen = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    route = ExpertRouting(24, 3, score="sigmoid")
    l = r(24)
    one, many = route.forward(l), route.forward(l[None])
    assert one[0].shape == (3,) and torch.equal(one[0], many[0][0]) and torch.equal(one[1], many[1][0])
    assert torch.equal(route.backward(l, *one, one[1]), route.backward(l[None], *many, many[1])[0])
    assert route.forward(l.new_empty(0, 24))[0].shape == (0, 3)
    assert route.backward(l.new_empty(0, 24), *route.forward(l.new_empty(0, 24)), l.new_empty(0, 3)).shape == (0, 24)
    head = I8Linear(40, 70, act="f32")
    head.load(r(70, 40))
    x = r(40)
    assert head.forward(x).shape == (70,) and torch.equal(head.forward(x), head.forward(x[None])[0])
    assert head.forward(x.new_empty(0, 40)).shape == (0, 70)
    for V in (300, 9000):
        sampler = Sampler(V)
        l, u = r(V), torch.rand((), generator=gen, device="cuda")
        one, many = sampler.forward(l, u, top_p=0.9), sampler.forward(l[None], u[None], top_p=0.9)
        assert one[0].shape == () and torch.equal(one[0], many[0][0]) and torch.equal(one[1], many[1][0])
        assert sampler.forward(l.new_empty(0, V), u.new_empty(0))[0].shape == (0,)


@pytest.mark.parametrize("E,k", [(80, 4), (200, 8)])
def test_training_by_a_rule_with_many_experts(E, k):
    """Forward, backward and the loads of a layer of more than 64 experts, against the layer in 64 bits."""
    from test_gpu_layer_routing import of
    c = Case(128, 64, E, k, "f32", "f32")
    r = rule(E, k, score="sigmoid", groups=8, top_groups=4)
    c.op.set_routing(r, balance=0.1)
    N = 300
    x = c.x(N)
    y = c.op.forward(x, train=True)
    idx, w, on = of(r, c.logits(x), None)
    dout = torch.randn(N, 128, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    c.op.zero_grad()
    dx = c.op.backward(dout)
    xd, wr = x.double().requires_grad_(), c.wr.double().requires_grad_()
    s = torch.sigmoid(xd @ wr + c.br.double())
    chosen = s.gather(1, idx.cuda())
    want = c.experts(xd, idx.cuda(), chosen / (chosen.sum(1, keepdim=True) + 1e-20))
    counts = torch.bincount(idx.reshape(-1), minlength=E).double().cuda()
    loss = (want * dout.double()).sum() + (0.1 * E * counts / N / N * s).sum()
    loss.backward()
    assert rel(y, want.detach()) < 1e-5
    assert rel(dx, xd.grad) < 1e-5
    assert rel(c.op.get_gradients()[0], wr.grad) < 1e-5
