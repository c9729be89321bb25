"""mgpt_lm_loss_forward / mgpt_lm_loss_backward (mgpt_amd.loss.LMLoss) against
the formulas in 64 bits, and the gradients against differences of the loss.

Tolerances, u = 2^-24.  A logit is a sum of C products and a bias: within
  ez = (C + 2) u (sum |x w| + |b|).
A log-sum-exp carries its logits' largest ez, the exponentials' arguments (2 u
of at most the row's range of logits), a sum of under 256 roundings in a row
of partial sums and a logarithm: el = max ez + 2 u range + 256 u (1 + |lse|).
A probability is off by a factor within exp(+-(ez + el + 2 u |z - lse| + 4 u)), so d by
that of it, one rounding, and in bf16 half a step, 2^-8 of it; a product with d
adds the roundings of its sum, K u of its K terms, and in bf16 half a step.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
HALF = {"f32": 0.0, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


def inputs(N, C, V, act, bias=True, seed=1, xstd=1.0, wstd=None):
    gen = torch.Generator().manual_seed(seed)
    dt = torch.float32 if act == "f32" else torch.bfloat16
    x = (torch.randn(N, C, generator=gen) * xstd).to(dt)
    W = (torch.randn(V, C, generator=gen) * (wstd or 2.0 / C ** 0.5)).to(dt)
    b = torch.randn(V, generator=gen) if bias else None
    t = torch.randint(0, V, (N,), generator=gen, dtype=torch.int32)
    return x.cuda(), W.cuda(), None if b is None else b.cuda(), t.cuda()


def reference(x, W, b, t, g=None):
    """{name: (value, tolerance in fp32)} in 64 bits, on the inputs' device; g:
    per row the upstream gradient (None: of the mean)."""
    N, C = x.shape
    V = W.shape[0]
    xd, Wd, t = x.double(), W.double(), t.long()
    z = xd @ Wd.t()
    amp = xd.abs() @ Wd.abs().t()
    if b is not None:
        z = z + b.double()
        amp = amp + b.double().abs()
    ez = (C + 2) * U * torch.nan_to_num(amp, posinf=0.0)
    lse = torch.logsumexp(z, 1)
    fin = torch.where(torch.isfinite(z), z, lse[:, None])
    el = ez.amax(1) + 2 * U * (fin.amax(1) - fin.amin(1)) + 256 * U * (1 + lse.abs())
    has = (t >= 0) & (t < V)
    tc = t.clamp(0, V - 1)
    loss = torch.where(has, lse - z.gather(1, tc[:, None])[:, 0], torch.zeros_like(lse))
    count = int(has.sum())
    eloss = torch.where(has, 2 * el + U * loss.abs(), torch.zeros_like(el))
    out = {"loss": (loss, eloss), "lse": (lse, el)}
    mean = loss.sum() / max(count, 1)
    out["mean"] = (torch.stack([mean, mean.new_tensor(float(count))]),
                   torch.stack([eloss.sum() / max(count, 1) + U * mean.abs(), mean.new_tensor(0.0)]))
    g = torch.full_like(lse, 1 / max(count, 1)) if g is None else g.double()
    g = torch.where(has, g, torch.zeros_like(g))
    p = (z - lse[:, None]).exp()
    rel = torch.expm1(ez + el[:, None] + 2 * U * (fin - lse[:, None]).abs() + 4 * U)
    d = p.clone()
    d.scatter_add_(1, tc[:, None], -torch.ones_like(lse)[:, None])
    ed = (p * rel + 3 * U * d.abs()) * g.abs()[:, None]
    d = d * g[:, None]
    ed = torch.where(has[:, None], ed, torch.zeros_like(ed))
    h = HALF["bf16" if x.dtype == torch.bfloat16 else "f32"]
    out["db"] = (d.sum(0), ed.sum(0) + (N + 4) * U * d.abs().sum(0))
    ed = ed + h * (d.abs() + ed)
    for name, a, ea, w, k in (("dx", d, ed, Wd, V), ("dW", d.t(), ed.t(), xd, N)):
        val = a @ w
        tol = ea @ w.abs() + (k + 8) * U * (a.abs() @ w.abs())
        out[name] = (val, tol + h * (val.abs() + tol))
    return out


def check(got, ref):
    for k, v in got.items():
        want, tol = ref[k]
        v = v.double()
        err = (v - want).abs()
        ok = (err <= tol + 1e-37) | ((v == want) & torch.isinf(want))
        assert ok.all(), (k, float((err / (tol + 1e-300)).max()), int((~ok).sum()))


def run(x, W, b, t, act, dloss=None, dmean=None):
    from mgpt_amd.loss import LMLoss
    op = LMLoss(x.shape[-1], W.shape[0], act=act)
    loss, lse, mean = op.forward(x, W, t, bias=b)
    dx, dW, db = op.backward(x, W, t, lse, bias=b, dloss=dloss, dmean=dmean)
    torch.cuda.synchronize()
    out = {"loss": loss, "lse": lse, "mean": mean, "dx": dx, "dW": dW}
    if db is not None:
        out["db"] = db
    return out


SHAPES = [(1, 16, 1), (1, 64, 16), (2, 1, 5), (3, 70, 33), (64, 128, 256), (65, 129, 257), (130, 64, 1000),
          (300, 500, 2003), (257, 320, 4099), (1030, 96, 700), (31, 2048, 300), (2100, 64, 4100), (513, 72, 129)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,V", SHAPES)
def test_loss_and_gradients(N, C, V, act):
    print(N, C, V, act, flush=True)
    x, W, b, t = inputs(N, C, V, act, bias=N % 2 == 1)
    if N > 8:   # rows without a target
        t[3], t[N // 2], t[N - 1] = -1, V, -2 ** 31
    check(run(x, W, b, t, act), reference(x, W, b, t))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,V", [(8192, 1024, 300), (8192, 1024, 2048), (256, 64, 33000)])
def test_large_tiles_and_split_contractions(N, C, V, act):
    print(N, C, V, act, flush=True)
    x, W, b, t = inputs(N, C, V, act)
    check(run(x, W, b, t, act), reference(x, W, b, t))


# Shapes of few tiles: every tile size with one tile a CU and with several, the gradients
# stored whole, by odd rows and in parts.
TILES = [(1, 8, 34875), (4327, 8, 2), (17916, 8, 2), (69, 8, 43707), (132, 8, 51576), (1, 1496, 1636), (5377, 1496, 3),
         (1065, 3600, 4), (1, 88, 8874), (1, 136, 53557), (1, 400, 27252), (1, 118, 8818), (2, 1572, 2468),
         (1, 12, 20526), (1, 131, 56687), (1, 75, 9109), (7, 3673, 1039), (1, 177, 58058), (1, 3280, 1272),
         (1, 3222, 2031), (1, 3348, 5455), (1, 3589, 11708), (943, 3385, 73), (216, 8, 16491), (17706, 135, 381),
         (4535, 72, 3396), (4435, 152, 11982), (40, 32, 30), (500, 64, 32), (4119, 3024, 2), (3302, 3783, 2),
         (3458, 3536, 2), (12841, 897, 2), (300, 1024, 20000), (300, 1025, 20000)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,V", TILES)
def test_tile_sizes(N, C, V, act):
    print(N, C, V, act, flush=True)
    x, W, b, t = inputs(N, C, V, act, bias=(N + C + V) % 2 == 1)
    check(run(x, W, b, t, act), reference(x, W, b, t))


@pytest.mark.parametrize("N,V,act", [(70000, 4200, "bf16"), (70001, 2100, "f32")])
def test_several_pieces_of_the_vocabulary(N, V, act):
    """More rows than one piece of the vocabulary has room for: the pieces'
    d W_piece add up."""
    print(N, V, act, flush=True)
    x, W, b, t = inputs(N, 64, V, act)
    check(run(x, W, b, t, act), reference(x, W, b, t))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_upstream_gradients(act):
    x, W, b, t = inputs(200, 96, 500, act)
    t[::7] = -1
    g = torch.randn(200, generator=torch.Generator().manual_seed(2)).cuda()
    g[5] = 0
    got = run(x, W, b, t, act, dloss=g)
    check(got, reference(x, W, b, t, g))
    m = torch.tensor([3.5], device="cuda")
    has = ((t >= 0) & (t < 500)).sum()
    # (the quotient's own rounding is one more of d's three)
    check(run(x, W, b, t, act, dmean=m), reference(x, W, b, t, torch.full_like(g, 3.5) / has))


def test_no_row_has_a_target():
    x, W, b, t = inputs(70, 64, 100, "bf16")
    t.fill_(-1)
    got = run(x, W, b, t, "bf16")
    check(got, reference(x, W, b, t))
    for k in ("loss", "mean", "dx", "dW", "db"):
        assert not got[k].any(), k


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min])
def test_masked_columns_and_large_logits(act, low):
    """Vocabulary entries masked by their bias get no probability and no
    gradient; logits of some hundreds neither overflow nor lose the sums."""
    x, W, b, t = inputs(140, 64, 400, act, xstd=20.0, wstd=2.0)
    b[5::3] = low
    t = (t // 3 * 3 + 3).clamp(max=399).int()     # columns 3, 6, ..: not masked
    got = run(x, W, b, t, act)
    keep = torch.ones(400, dtype=torch.bool, device="cuda")
    keep[5::3] = False
    assert not got["dW"][~keep].any() and not got["db"][~keep].any()
    at = torch.cumsum(keep.int(), 0) - 1
    ref = reference(x, W[keep], b[keep], at[t.long()].int())
    got = {k: v[keep] if k in ("dW", "db") else v for k, v in got.items()}
    check(got, ref)


def test_every_logit_at_the_lowest_value():
    """A row's logits all the type's lowest: the softmax is uniform."""
    x = torch.zeros(3, 64, device="cuda")
    W = torch.zeros(130, 64, device="cuda")
    b = torch.full((130,), torch.finfo(torch.float32).min, device="cuda")
    t = torch.tensor([0, 129, 64], dtype=torch.int32, device="cuda")
    got = run(x, W, b, t, "f32")
    assert (got["lse"] == b[0]).all()   # log 130 is far below half a step there
    assert (got["loss"] == 0).all()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_row_without_a_target_may_hold_anything(act, value):
    """Padding that is not finite changes no gradient and no other row."""
    x, W, b, t = inputs(100, 64, 300, act)
    t[17], t[99] = -1, 300
    clean = run(x, W, b, t, act)
    x2 = x.clone()
    x2[17, 5] = value
    x2[99] = value
    got = run(x2, W, b, t, act)
    assert not torch.isfinite(got["lse"][17]) and got["loss"][17] == 0 and got["loss"][99] == 0
    rows = torch.ones(100, dtype=torch.bool, device="cuda")
    rows[17] = rows[99] = False
    for k in ("loss", "lse", "dx"):
        assert torch.equal(got[k][rows], clean[k][rows]), k
    for k in ("mean", "dW", "db"):
        assert torch.equal(got[k], clean[k]), k
    assert not got["dx"][~rows].any()


def test_a_row_with_a_target_that_is_not_finite():
    """Its loss is NaN, the others' are as before."""
    x, W, b, t = inputs(100, 64, 300, "bf16")
    clean = run(x, W, b, t, "bf16")
    x2 = x.clone()
    x2[17, 5] = float("nan")
    got = run(x2, W, b, t, "bf16")
    rows = torch.arange(100, device="cuda") != 17
    assert torch.isnan(got["loss"][17]) and torch.equal(got["loss"][rows], clean["loss"][rows])
    assert torch.equal(got["dx"][rows], clean["dx"][rows])


def test_gradients_are_the_losses_differences():
    """Along random directions, central differences of the mean loss in 64 bits:
    with steps of 1e-5 their error is under 1e-8; the gradients' tolerance is
    reference()'s, summed along the direction."""
    x, W, b, t = inputs(40, 24, 70, "f32")
    t[4] = -1
    got = run(x, W, b, t, "f32")
    ref = reference(x, W, b, t)
    gen = torch.Generator().manual_seed(4)
    for name, src in (("dx", x), ("dW", W), ("db", b)):
        v = torch.randn(src.shape, generator=gen, dtype=torch.float64).cuda()
        ends = []
        for sign in (1, -1):
            a = {"dx": x.double(), "dW": W.double(), "db": b.double()}
            a[name] = a[name] + sign * 1e-5 * v
            ends.append(reference(a["dx"], a["dW"], a["db"], t)["mean"][0][0])
        diff = float(ends[0] - ends[1]) / 2e-5
        along = float((got[name].double() * v).sum())
        assert abs(diff - along) <= 1e-8 + float((ref[name][1] * v.abs()).sum()), (name, diff, along)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_tensors_at_odd_addresses(act):
    x, W, b, t = inputs(90, 128, 300, act)
    want = run(x, W, b, t, act)

    def moved(v):
        buf = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")
        out = buf[1:].view(v.shape)
        out.copy_(v)
        return out

    got = run(moved(x), moved(W), moved(b), moved(t), act)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_some_gradients_only():
    from mgpt_amd.loss import LMLoss
    x, W, b, t = inputs(150, 64, 333, "bf16")
    want = run(x, W, b, t, "bf16")
    op = LMLoss(64, 333)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        got = op.backward(x, W, t, want["lse"], bias=b, need=need)
        for g, k, n in zip(got, ("dx", "dW", "db"), need):
            assert (g is None) == (not n)
            if n:
                assert torch.equal(g, want[k])


def test_same_bits_on_another_stream_and_in_a_graph():
    from mgpt_amd.loss import LMLoss
    x, W, b, t = inputs(700, 192, 3001, "bf16")
    want = run(x, W, b, t, "bf16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(x, W, b, t, "bf16")
    op = LMLoss(192, 3001)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse, mean = op.forward(x, W, t, bias=b)
        dx, dW, db = op.backward(x, W, t, lse, bias=b)
    for k in want:
        assert torch.equal(want[k], again[k]), k
    for _ in range(3):
        for v in (loss, lse, mean, dx, dW, db):
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for k, v in zip(("loss", "lse", "mean", "dx", "dW", "db"), (loss, lse, mean, dx, dW, db)):
            assert torch.equal(want[k], v), k
        run(x[:300].contiguous(), W, b, t[:300].contiguous(), "bf16")


def test_two_calls_at_once():
    """Calls in flight on two streams have workspaces of their own."""
    x, W, b, t = inputs(900, 256, 5000, "bf16")
    want = run(x, W, b, t, "bf16")
    x2 = x.flip(0).contiguous()
    want2 = run(x2, W, b, t, "bf16")
    from mgpt_amd.loss import LMLoss
    op = LMLoss(256, 5000)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for st, xi in zip(s, (x, x2)):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            loss, lse, mean = op.forward(xi, W, t, bias=b)
            got.append((loss, *op.backward(xi, W, t, lse, bias=b)))
    torch.cuda.synchronize()
    for g, w in zip(got, (want, want2)):
        for v, k in zip(g, ("loss", "dx", "dW", "db")):
            assert torch.equal(v, w[k]), k


def test_no_tokens():
    for act in ("f32", "bf16"):
        x, W, b, t = inputs(1, 7, 9, act)
        got = run(x[:0], W, b, t[:0], act)
        assert got["loss"].shape == (0,) and not got["mean"].any()
        assert not got["dW"].any() and not got["db"].any()
