"""MoELayer(weights="i8") against its formula in 64 bits: rows quantised as gathered, gate and
up, h = silu(g) u, h quantised in turn, down, weighted.

What the device's h differs from the exact one by (for bf16 the 20 bits it is held in, at most 2^-16 of a group's
largest; some 2^-20 of g and u) moves it across a border between two integers with that probability, in integer
steps up to 2 127 2^-16 + 127 2^-18 < 0.005.  An output's error is a sum over k of such steps, each of at most b = 127 sh sd and with a
variance of at most 0.005 (sh qd_k sd)^2, v in sum: by Bernstein's inequality it passes t = c b + sqrt((c b)^2 + 6 c v) with
a probability of 2 exp(-3 c); c = 20 / 3 makes that 4e-9 of an output.  Beside t the tolerance has 2^-7 of the summed
magnitudes for the two roundings to bf16 (2^-8 each) of outputs and sum, and the float sums' 2^-18.  (The first form of this,
6 standard deviations, took the sum for a normal one; with 64 hidden units one row in five hundred has two steps.)
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def quantised(a):
    top = a.double().abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.round(a.double() * (127 / top)), torch.zeros(()).double().to(a.device))
    return q, (top / 127).squeeze(-1)


class Layer:
    def __init__(self, C, H, E, k, act="bf16", seed=1):
        from mgpt_amd.moe import MoELayer
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.C, self.H, self.E, self.k = C, H, E, k
        self.wr, self.br = r(C, E) * 0.1, r(E) * 0.1
        self.W = {n: r(E, a, b) / a ** 0.5 for n, a, b in (("g", C, H), ("u", C, H), ("d", H, C))}
        self.b = {n: r(E, self.W[n].shape[2]) * 0.1 for n in "gud"}
        self.op = MoELayer(C, H, E, k, act=act, weights="i8")
        params = [self.wr, self.br]
        for e in range(E):
            for n in "gud":
                params += [self.W[n][e], self.b[n][e]]
        self.op.load_parameters(params)
        self.dt = torch.float32 if act == "f32" else torch.bfloat16

    def inputs(self, N, seed=2, skew=0.3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(N, self.C, generator=gen, device="cuda").to(self.dt)
        s = torch.randn(N, self.E, generator=gen, device="cuda")
        s = s + torch.randn(self.E, generator=gen, device="cuda") * skew
        top, idx = s.topk(self.k, 1)
        return x, idx.int(), torch.softmax(top, 1)

    def expert(self, e, x):
        """(output, its steps' largest size, their variance) of rows x."""
        def product(a, n):
            q, sa = quantised(a)
            w, sw = quantised(self.W[n][e].t())
            unit = sa[:, None] * sw
            return (q @ w.t()) * unit + self.b[n][e].double(), 127 * unit, 0.005 * unit ** 2 * (w * w).sum(1)
        h = torch.nn.functional.silu(product(x, "g")[0]) * product(x, "u")[0]
        return product(h, "d")

    def check(self, y, x, idx, w, base=None):
        want = torch.zeros(x.shape[0], self.C, dtype=torch.float64, device="cuda")
        mag, var, step = torch.zeros_like(want), torch.zeros_like(want), torch.zeros_like(want)
        for e in range(self.E):
            t, j = (idx == e).nonzero(as_tuple=True)
            if t.numel():
                o, b, v = self.expert(e, x[t].double())
                p = w[t, j].double()[:, None]
                want.index_add_(0, t, o * p)
                mag.index_add_(0, t, (o * p).abs())
                var.index_add_(0, t, v * p * p)
                step.index_add_(0, t, b * p)      # (at least each expert's own)
        if base is not None:
            want, mag = want + base.double(), mag + base.double().abs()
        step *= 20 / 3
        tol = step + (step ** 2 + 40 * var).sqrt() + 2.0 ** -7 * mag + 2.0 ** -18 * mag.amax(1, keepdim=True)
        bad = (y.double() - want).abs() > tol
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4], y[bad][:4], want[bad][:4])
        # and on the whole far nearer: the two roundings alone
        assert ((y.double() - want).norm() / want.norm()).item() < 0.005
        return want


# decode (one and two row blocks a segment, contractions split), 128 x 128 and 256 x 256 tiles; odd widths,
# experts without rows, more than 64 of them
CASES = [(1, 64, 96, 4, 2), (3, 200, 100, 8, 8), (24, 512, 300, 8, 2), (64, 1024, 704, 64, 8), (33, 96, 2048, 2, 1),
         (100, 512, 1376, 16, 2), (300, 256, 512, 4, 2), (700, 1000, 333, 6, 3), (2000, 640, 1408, 8, 2),
         (5000, 512, 1376, 8, 2), (600, 128, 256, 96, 8), (4000, 256, 384, 130, 4), (9000, 64, 64, 3, 1)]


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("N,C,H,E,k", CASES)
def test_given_routing(N, C, H, E, k, act):
    L = Layer(C, H, E, k, act)
    x, idx, w = L.inputs(N)
    y = L.op.forward_routed(x, idx, w)
    L.check(y, x, idx, w)
    assert torch.equal(y, L.op.forward_routed(x, idx, w))
    r = L.op.routing()
    assert torch.equal(r["topk_idx"], idx) and torch.equal(r["counts"].long(), torch.bincount(idx.view(-1), minlength=E))


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_the_layers_own_router_and_block(act):
    for N in (50, 900):
        L = Layer(256, 512, 8, 2, act)
        x = L.inputs(N)[0]
        y = L.op.forward(x)
        r = L.op.routing()
        L.check(y, x, r["topk_idx"], r["topk_p"])
        gamma = 1 + 0.1 * torch.randn(256, device="cuda")
        z = L.op.forward_block(x, gamma)
        r = L.op.routing()
        n = x.float() * L.op.rstd()[:, None] * gamma
        L.check(z, n, r["topk_idx"], r["topk_p"], base=x)


def test_all_rows_to_one_expert_and_ids_out_of_range():
    for N in (20, 700):
        L = Layer(128, 256, 8, 4)
        x, idx, w = L.inputs(N)
        idx[:] = 5                           # four times the same expert
        L.check(L.op.forward_routed(x, idx, w), x, idx, w)
        x, idx, w = L.inputs(N)
        bad = idx.clone()
        bad[::3, 1] = -1
        bad[1::3, 0] = 8
        bad[2::3, 2] = 2 ** 31 - 1
        v = torch.where((bad >= 0) & (bad < 8), w, torch.zeros_like(w))
        y = L.op.forward_routed(x, bad, w)
        L.check(y, x, torch.where(v != 0, bad, torch.zeros_like(bad)), v)


def test_rows_that_are_not_finite_and_hidden_units_of_any_size():
    L = Layer(128, 256, 4, 2)
    for N in (30, 600):
        x, idx, w = L.inputs(N)
        clean = L.op.forward_routed(x, idx, w)
        for bad in (float("nan"), float("inf")):
            z = x.clone()
            z[7, 3] = bad
            y = L.op.forward_routed(z, idx, w)
            assert y[7].isnan().all()
            keep = [i for i in range(N) if i != 7]
            assert torch.equal(y[keep], clean[keep])
        z = x.clone()
        z[3] = 0
        z[4] *= 1e-20
        z[5] *= 1e12
        L.check(L.op.forward_routed(z, idx, w), z, idx, w)


def test_refusals():
    L = Layer(64, 64, 4, 2)
    x, idx, w = L.inputs(10)
    for bad in (lambda: L.op.forward_routed(x.float(), idx, w), lambda: L.op.forward_routed(x, idx.long(), w),
                lambda: L.op.forward_routed(x, idx[:, :1], w), lambda: L.op.forward_routed(x, idx, w.double()),
                lambda: L.op.forward_routed(x, idx.t().contiguous().t(), w)):
        with pytest.raises(ValueError):
            bad()
    from mgpt_amd import capi
    with pytest.raises(capi.MoEError):
        L.op.forward(x, train=True)
    assert L.op.forward_routed(x[:0], idx[:0], w[:0]).shape == (0, 64)


def test_replayed_graph():
    for N in (40, 500):
        L = Layer(256, 384, 8, 2)
        x, idx, w = L.inputs(N)
        L.op.forward_routed(x, idx, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = L.op.forward_routed(x, idx, w)
        for seed in (3, 4, 5):
            nx, ni, nw = L.inputs(N, seed)
            x.copy_(nx), idx.copy_(ni), w.copy_(nw)
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            assert torch.equal(got, L.op.forward_routed(x, idx, w))
