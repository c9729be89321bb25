"""Places of a routing that no expert takes: ids out of range in MoELayer.forward_routed, weights of 0, and what a rule
(set_routing) fills up with where fewer than k experts take part.  They count for nothing: not in y, whatever is in x,
not in the experts' counts, and not in the balance loss.  Bars as in test_gpu_layer_routing.py: of an output the bar is on
each term's size, so that on their sum's it is at most that of the sizes' sum, which the sum may be far below (three
terms of one token under fp8 weights)."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_layer_routing import BAR, Case, of, rel, rule  # noqa: E402

INF, NAN = float("inf"), float("nan")
KINDS = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "fp8"), ("f32", "fp8"), ("f32", "bf16"), ("bf16", "i8"), ("f32", "i8")]


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def sizes(c, x, idx, w):
    """The sum over the places of their terms' norms."""
    return sum(c.experts(x.double(), idx[:, j:j + 1], w[:, j:j + 1].double()).norm() for j in range(idx.shape[1]))


@pytest.mark.parametrize("act,weights", KINDS)
@pytest.mark.parametrize("E,k,C", [(8, 4, 128), (8, 2, 64), (64, 8, 256), (80, 2, 192), (6, 1, 100)])
def test_ids_out_of_range_and_weights_of_zero(E, k, C, act, weights):
    c = Case(C, 128, E, k, act, weights)
    for N in (1, 20, 64, 300, 1500):
        gen = torch.Generator(device="cuda").manual_seed(N)
        x = c.x(N)
        idx = torch.rand(N, E, generator=gen, device="cuda").topk(k, 1)[1].int()
        w = torch.rand(N, k, generator=gen, device="cuda") + 0.1
        none = torch.rand(N, k, generator=gen, device="cuda") < 0.3
        none[::3] = True                     # tokens of no expert at all
        x[::3, 5] = NAN
        x[::6, 7] = INF
        out = torch.where(none, torch.where(idx % 2 == 0, -1, E + 3).int(), idx)
        zero = torch.where(none, torch.zeros_like(w), w)
        y = c.op.forward_routed(x, out, w)
        r = c.op.routing()
        assert torch.equal(r["counts"].long(), torch.bincount(idx[~none].long(), minlength=E))
        assert (y[::3] == 0).all()
        live = torch.ones(N, dtype=torch.bool, device="cuda")
        live[::3] = False
        if live.any():
            want = c.experts(x[live].double(), torch.where(none, -1, idx)[live], w[live].double())
            assert (y[live].double() - want).norm() <= BAR[weights] * sizes(c, x[live], torch.where(none, -1, idx)[live], w[live])
        assert same(c.op.forward_routed(x, idx, zero), y)
        assert same(c.op.forward_routed(x, torch.full_like(idx, -1), w), torch.zeros_like(y))


@pytest.mark.parametrize("act,weights", KINDS)
@pytest.mark.parametrize("E,k,groups,C", [(32, 8, 8, 64), (12, 4, 4, 128), (96, 8, 32, 64), (8, 2, 8, 64)])
def test_rules_that_leave_fewer(E, k, groups, C, act, weights):
    """One group of E / groups experts takes part."""
    c = Case(C, 128, E, k, act, weights)
    left = E // groups
    for kw in (dict(score="sigmoid"), dict(score="softmax", renormalise=False)):
        op = rule(E, k, groups=groups, top_groups=1, group_best=1, **kw)
        c.op.set_routing(op)
        for N in (1, 40, 700):
            x = c.x(N)
            y = c.op.forward(x)
            r = c.op.routing()
            idx, w, on = of(op, c.logits(x), None)
            idx, w, on = idx.cuda(), w.cuda(), on.cuda().bool()
            assert int(on.sum()) == N * min(k, left)
            assert torch.equal(r["counts"].long(), torch.bincount(idx[on], minlength=E))
            assert torch.equal(r["topk_idx"].long(), torch.where(on, idx, torch.full_like(idx, -1)))
            taken = torch.where(on, idx, torch.full_like(idx, -1))
            assert (y.double() - c.experts(x.double(), taken, w)).norm() <= BAR[weights] * sizes(c, x, taken, w)
            # the same from the rule alone, whose fillers have weight 0
            i, v = op.forward(c.logits(x))
            assert torch.equal(c.op.forward_routed(x, i, v), y)
        c.op.set_routing(None)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N", [60, 900])
@pytest.mark.parametrize("masked", [False, True])
def test_training_with_fewer_than_k(act, N, masked):
    """By groups, or by a bias of -infinity; the balance loss counts the experts that take part."""
    E, k, C, H, balance = 16, 4, 64, 96, 0.5
    c = Case(C, H, E, k, act, act)
    bias = None
    if masked:
        bias = torch.full((E,), -INF, device="cuda")
        bias[3::5] = torch.tensor([0.0, 0.05, -0.05], device="cuda")     # 3 of 16 experts
        op = rule(E, k, score="sigmoid")
    else:
        op = rule(E, k, score="softmax", groups=8, top_groups=1, scale=1.5)
    c.op.set_routing(op, bias=bias, balance=balance)
    x = c.x(N)
    dy = torch.randn(N, C, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(x.dtype)
    for again in range(2):
        c.op.reserve(N, train=True)
        c.op._ws.fill_(255 if again else 0)      # (what a workspace held before makes no difference: NaN, ids of -1)
        c.op.zero_grad()
        y = c.op.forward(x, train=True)
        dx = c.op.backward(dy)
        idx, _, on = of(op, c.logits(x), bias)
        idx, on = idx.cuda(), on.cuda().bool()
        assert not on.all()
        taken = torch.where(on, idx, torch.full_like(idx, -1))
        counts = torch.bincount(idx[on], minlength=E).double()
        assert torch.equal(c.op.routing()["counts"].double(), counts)
        xd = x.double().requires_grad_()
        leaves = [t.double().requires_grad_() for t in (c.wr, c.br, *c.W, *c.b)]
        l = xd @ leaves[0] + leaves[1]
        s = torch.softmax(l, 1) if op.config.score == 0 else torch.sigmoid(l)
        sel = s.gather(1, idx) * on
        w = sel * op.config.scale / (sel.sum(1, keepdim=True) + 1e-20)
        ref = c.experts(xd, taken, w, leaves[2:5], leaves[5:])
        assert rel(y, ref.detach()) < BAR[act]
        ((ref * dy.double()).sum() + (s * (balance * E * counts / N / N)).sum()).backward()
        assert rel(dx, xd.grad) < BAR[act]
        got = c.op.get_gradients()
        assert rel(got[0], leaves[0].grad) < BAR[act] and rel(got[1].view(-1), leaves[1].grad) < BAR[act]
        for i in range(3):
            gW = torch.stack([got[2 + 6 * e + 2 * i] for e in range(E)])
            gb = torch.stack([got[3 + 6 * e + 2 * i].view(-1) for e in range(E)])
            assert rel(gW, leaves[2 + i].grad) < BAR[act] and rel(gb, leaves[5 + i].grad) < BAR[act]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N", [1, 70, 1200])
def test_training_of_no_expert_at_all(act, N):
    """Every expert masked: y, dx and all gradients are 0, by the layer alone and in the block (y = x, dx = dy)."""
    E, k, C = 8, 2, 64
    c = Case(C, 96, E, k, act, act)
    c.op.set_routing(rule(E, k, score="sigmoid"), bias=torch.full((E,), -INF, device="cuda"), balance=0.5)
    x, gamma = c.x(N), torch.ones(C, device="cuda")
    dy = torch.randn(N, C, device="cuda").to(x.dtype)
    c.op.reserve(N, train=True)
    c.op._ws.fill_(255)
    c.op.zero_grad()
    y = c.op.forward(x, train=True)
    dx = c.op.backward(dy)
    assert (y == 0).all() and (dx == 0).all() and (c.op.routing()["counts"] == 0).all()
    assert all((g == 0).all() for g in c.op.get_gradients())
    out = torch.empty_like(x)
    c.op.forward_block_into(x, gamma, 1e-5, out, train=True)
    dx, dgamma = c.op.backward_block(dy)
    assert torch.equal(out, x) and torch.equal(dx, dy) and (dgamma == 0).all()
    assert all((g == 0).all() for g in c.op.get_gradients())


def test_replayed_graph():
    c = Case(64, 96, 8, 2, "bf16", "i8")
    for N in (30, 500):
        x = c.x(N)
        idx = torch.zeros(N, 2, dtype=torch.int32, device="cuda")
        w = torch.ones(N, 2, device="cuda")
        c.op.forward_routed(x, idx, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = c.op.forward_routed(x, idx, w)
        for seed in (3, 4, 5):
            gen = torch.Generator(device="cuda").manual_seed(seed)
            idx.copy_(torch.randint(-4, 8, (N, 2), generator=gen, device="cuda", dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            assert torch.equal(got, c.op.forward_routed(x, idx, w))
            assert (got[(idx < 0).all(1)] == 0).all()
