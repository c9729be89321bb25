"""Sampler (mgpt_sample) against its definition in 64 bits and whole numbers.

The tokens have to be equal.  (A weight next to half a unit may round to the other one in the device's
exponential: one part in 2^40, which moves a token with a probability of 2^-40 times the vocabulary.)  logp: the
logarithm in 64 bits, rounded once, 2^-24 of it, and 2^-40 of the sums' own rounding.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

INF = float("inf")
BIG = torch.finfo(torch.float32).max
UNITS = 2.0 ** 40


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def reference(logits, u, T, k, p, m):
    """(tokens, log-probabilities, kept) on the device, rows at a time; T, k, p, m: [B]."""
    B, V = logits.shape
    l = logits.float()
    l = torch.where(l.isnan(), torch.full_like(l, -INF), l.clamp(max=BIG))
    top = l.amax(1, keepdim=True)
    empty = (top == -INF).squeeze(1)
    greedy = ~(T > 0)
    sl, si = torch.sort(l, dim=1, descending=True, stable=True)
    Td = torch.where(greedy, torch.ones_like(T), T).double()[:, None]
    z = torch.where(sl > -INF, (sl.double() - top.double()) / Td, torch.full_like(sl, -INF).double())
    W = (z.exp() * UNITS).round()
    k = torch.where(k <= 0, torch.full_like(k, V), k)
    k = torch.where(greedy, torch.ones_like(k), k)
    first = torch.arange(V, device=l.device)[None] < k[:, None]
    Wk = torch.where(first, W, torch.zeros_like(W)).long()
    run = Wk.cumsum(1)
    pd = p.double()[:, None]
    keep = first & (((run - Wk).double() < pd * run[:, -1:].double()) | (pd >= 1))
    keep &= W >= m.double()[:, None] * UNITS
    keep[:, 0] = True
    mine = torch.zeros_like(Wk).scatter_(1, si, torch.where(keep, Wk, torch.zeros_like(Wk)))
    run = mine.cumsum(1)
    total = run[:, -1:]
    at = (run.double() <= u.clamp(min=0).double()[:, None] * total.double()).sum(1)
    at = torch.minimum(at, (run < total).sum(1)).clamp(max=V - 1)
    zt = (l.gather(1, at[:, None]).double() - top.double()) / Td
    logp = zt.squeeze(1) - (total.squeeze(1).double() / UNITS).log()
    at = torch.where(empty, torch.full_like(at, -1), at)
    logp = torch.where(empty, torch.full_like(logp, -INF), logp)
    return at.int(), logp, (mine > 0).sum(1)


def check(logits, u, T=1.0, k=0, p=1.0, m=0.0):
    from mgpt_amd.sampling import Sampler
    B, V = logits.shape
    op = Sampler(V, act="f32" if logits.dtype == torch.float32 else "bf16")
    rows = lambda v, dt: v if isinstance(v, torch.Tensor) else torch.full((B,), v, dtype=dt, device="cuda")  # noqa: E731
    f = torch.float32
    token, logp = op.forward(logits, u, temperature=T, top_k=k, top_p=p, min_p=m)
    rt, rl, kept = reference(logits, u, rows(T, f), rows(k, torch.int32), rows(p, f), rows(m, f))
    bad = token != rt
    assert not bad.any(), (bad.nonzero()[:4].tolist(), token[bad][:4].tolist(), rt[bad][:4].tolist(), kept[bad][:4].tolist())
    fine = rt >= 0
    assert ((logp - rl).abs()[fine] <= 2.0 ** -24 * rl.abs()[fine] + 2.0 ** -38).all()
    assert (logp[~fine] == -INF).all()
    again = op.forward(logits, u, temperature=T, top_k=k, top_p=p, min_p=m)
    assert torch.equal(token, again[0]) and torch.equal(logp, again[1])
    return token, kept


def inputs(B, V, act, seed=1, std=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    l = (torch.randn(B, V, generator=gen, device="cuda") * std).to(torch.float32 if act == "f32" else torch.bfloat16)
    return l, torch.rand(B, generator=gen, device="cuda")


FILTERS = [dict(), dict(k=1), dict(k=7), dict(k=50, p=0.9), dict(k=900), dict(p=0.95), dict(p=0.3, T=0.7), dict(m=0.05),
           dict(p=0.8, m=0.02, T=1.4), dict(k=200, p=0.97, m=0.001, T=3.0), dict(T=0.0), dict(p=0.0), dict(m=1.0), dict(m=1.5),
           dict(k=5000, p=0.999), dict(T=50.0, p=0.6), dict(T=0.01, p=0.9)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 3, 31, 100, 257, 1000, 4099, 20000, 50257, 131072])
def test_filters(V, act):
    for i, f in enumerate(FILTERS):
        l, u = inputs(17, V, act, seed=V + i)
        check(l, u, **f)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_rows_with_their_own_parameters(act):
    B, V = 96, 7001
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda: torch.rand(B, generator=gen, device="cuda")  # noqa: E731
    l, u = inputs(B, V, act)
    T = r() * 2
    T[::9] = 0
    k = torch.randint(-1, 2000, (B,), generator=gen, device="cuda", dtype=torch.int32)
    k[::5] = 0
    p, m = r() * 1.2, r() * 0.1
    m[::3] = 0
    check(l, u, T, k, p, m)
    # one of each kind given as a number
    check(l, u, T, 40, p, 0.0)
    check(l, u, 0.8, k, 0.9, m)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_ties(act):
    """Equal logits are cut at the lowest ids: few different values, all equal, more than a list takes."""
    for V in (300, 9000, 70000):
        gen = torch.Generator(device="cuda").manual_seed(V)
        u = torch.rand(12, generator=gen, device="cuda")
        l = torch.randint(-3, 3, (12, V), generator=gen, device="cuda").to(inputs(1, 1, act)[0].dtype)
        l[0] = 0
        l[1] = -5.5
        l[2, ::2] = -0.0
        for f in (dict(k=3), dict(k=V // 2), dict(k=V - 1), dict(p=0.5), dict(p=0.9), dict(k=V // 3, p=0.9), dict(m=0.3),
                  dict(k=V // 2, p=0.999, m=0.01), dict(T=0.0), dict()):
            check(l, u, **f)


def test_masks_infinities_and_far_logits():
    for V in (50, 3000):
        l, u = inputs(24, V, "f32")
        l[0] = -INF
        l[1, 1:] = -INF
        l[2, :-1] = -INF
        l[3] = float("nan")
        l[4, ::2] = float("nan")
        l[5, 7] = INF
        l[6, 5:9] = INF
        l[7] = INF
        l[8] = -BIG
        l[9, 3] = BIG
        l[10] *= 1e30
        l[11] *= 1e-30
        l[12, ::3] = -INF
        l[13] = -INF
        l[13, 9] = -BIG
        l[14] += 1e6
        l[15] -= 3e4
        for f in FILTERS:
            check(l, u, **f)
        for T in (1e-30, 1e-42, 1e30, INF):
            check(l[11:13].contiguous(), u[:2].contiguous(), T=T, k=11)
            check(l[16:].contiguous(), u[16:].contiguous(), T=T, p=0.7)


def test_random_numbers_at_the_ends():
    l, _ = inputs(6, 1000, "f32")
    u = torch.tensor([0.0, 1.0, 1 - 2.0 ** -24, 2.0 ** -149, 0.5, 2.0], device="cuda")
    for f in FILTERS:
        check(l, u, **f)


def test_the_draw_follows_the_distribution():
    """Evenly spread random numbers reach each token as often as its probability says, to one."""
    from mgpt_amd.sampling import Sampler
    B, V = 4096, 37
    l = inputs(1, V, "f32")[0].expand(B, V).contiguous()
    u = (torch.arange(B, device="cuda") + 0.5) / B
    token, logp = Sampler(V).forward(l, u, temperature=0.9, top_k=20)
    p = torch.zeros(V, device="cuda", dtype=torch.float64)
    top, at = l[0].double().topk(20)
    p[at] = torch.softmax(top / 0.9, 0)
    n = torch.bincount(token.long(), minlength=V)
    assert ((n - p * B).abs() <= 1).all()
    assert ((logp.double().exp() - p[token.long()]).abs() < 1e-6).all()


def test_the_largest_rows_and_offsets_past_32_bits():
    V = 1 << 20
    for act in ("f32", "bf16"):
        l, u = inputs(3, V, act)
        for f in (dict(), dict(k=40), dict(p=0.9), dict(k=100000, p=0.99, m=1e-5)):
            check(l, u, **f)
        check(torch.zeros_like(l), u, k=700000, p=0.7)
    B = 2100
    l = torch.zeros(B, V, dtype=torch.bfloat16, device="cuda")
    tail, u = inputs(4, V, "bf16")
    l[-4:] = tail
    uu = torch.full((B,), 0.25, device="cuda")
    uu[-4:] = u
    from mgpt_amd.sampling import Sampler
    token, _ = Sampler(V, act="bf16").forward(l, uu, top_p=0.9)
    want, _ = Sampler(V, act="bf16").forward(tail, u, top_p=0.9)
    assert torch.equal(token[-4:], want)


def test_rows_at_any_element_streams_graphs():
    from mgpt_amd.sampling import Sampler
    V = 5003
    for act in ("f32", "bf16"):
        l, u = inputs(9, V, act)
        op = Sampler(V, act=act)
        want = op.forward(l, u, top_p=0.9)
        flat = torch.empty(9 * V + 8, dtype=l.dtype, device="cuda")
        for off in (0, 1, 3, 7):
            v = flat[off:off + 9 * V].view(9, V)
            v.copy_(l)
            got = op.forward(v, u, top_p=0.9)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = op.forward(l.view(3, 3, V), u.view(3, 3), top_p=0.9)
        assert torch.equal(got[0].view(-1), want[0])
        assert op.forward(l[:0], u[:0])[0].shape == (0,)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got = op.forward(l, u, top_p=0.9)
        st.synchronize()
        assert torch.equal(got[0], want[0])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            token, logp = op.forward(l, u, top_k=30, top_p=0.9)
        for seed in (5, 6, 7):
            nl, nu = inputs(9, V, act, seed)
            l.copy_(nl), u.copy_(nu)
            graph.replay()
            torch.cuda.synchronize()
            got = op.forward(l, u, top_k=30, top_p=0.9)
            assert torch.equal(got[0], token) and torch.equal(got[1], logp)


@pytest.mark.parametrize("V", [8193, 20011])
def test_masks_and_far_logits_in_long_rows(V):
    l, u = inputs(20, V, "f32", seed=V)
    l[0] = -INF
    l[1, 1:] = -INF
    l[2, :-1] = -INF
    l[3] = float("nan")
    l[4, ::2] = float("nan")
    l[5, 7] = INF
    l[6, 5::900] = INF
    l[7] = INF
    l[8] = -BIG
    l[9, V - 3] = BIG
    l[10] *= 1e30
    l[11] *= 1e-30
    l[12, ::3] = -INF
    l[13] = -INF
    l[13, 9] = -BIG
    l[14] += 1e6
    l[15, ::2] = 0.0
    l[15, 1::2] = -0.0
    for f in FILTERS:
        check(l, u, **f)
    for T in (1e-30, 1e-42, 1e30, INF):
        check(l[11:13].contiguous(), u[:2].contiguous(), T=T, k=11)
        check(l[15:].contiguous(), u[15:].contiguous(), T=T, p=0.7)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_long_rows_with_their_own_parameters(act):
    """More rows than a launch takes; lists of few and of many, none, and rows that settle at once, side by side."""
    B, V = 2077, 9001
    gen = torch.Generator(device="cuda").manual_seed(4)
    r = lambda: torch.rand(B, generator=gen, device="cuda")  # noqa: E731
    l, u = inputs(B, V, act)
    T = r() * 2
    T[::9] = 0
    k = torch.randint(-1, 1500, (B,), generator=gen, device="cuda", dtype=torch.int32)
    k[::5] = 0
    k[1::5] %= 60
    p, m = r() * 1.2, r() * 0.1
    m[::3] = 0
    check(l, u, T, k, p, m)
    check(l, u, 0.8, 0, p, m)


def test_the_list_takes_no_more():
    """Rows whose bin holds 4096 logits, one fewer and one more, and top_k at the list's own ends."""
    V = 30000
    l, u = inputs(8, V, "f32", std=0.5)
    l.clamp_(max=3.0)
    for row, n in enumerate((4095, 4096, 4097, 255, 256, 257, 1024, 12000)):
        l[row, 100:100 + n] = 5.0
    for k in (1, 2, 255, 256, 257, 1023, 1024, 1025, 4096, 4097, V - 1, V, V + 5):
        check(l, u, k=k)
        check(l, u, k=k, p=0.5, m=0.01)
    check(l, u, p=0.4)
    check(l, u, p=0.9, T=0.5)


def test_long_rows_streams_graphs():
    from mgpt_amd.sampling import Sampler
    V = 20001
    op = Sampler(V, act="bf16")
    l, u = inputs(9, V, "bf16")
    kinds = (dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.9), dict(top_k=3000))
    op.forward(l, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [op.forward(l, u, **f) for f in kinds]
    for seed in (5, 6, 7):
        nl, nu = inputs(9, V, "bf16", seed)
        l.copy_(nl), u.copy_(nu)
        graph.replay()
        torch.cuda.synchronize()
        for f, (token, logp) in zip(kinds, out):
            got = op.forward(l, u, **f)
            assert torch.equal(got[0], token) and torch.equal(got[1], logp)
    # two streams at once, a workspace each
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = [op.forward(l, u, **f) for f in kinds]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                got.append([op.forward(l, u, **f) for f in kinds])
    torch.cuda.synchronize()
    assert all(torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) for g in got for a, b in zip(g, want))


def test_bf16_values_of_any_size_in_long_rows():
    """Values inside and outside 2^-8 to 2^8, which are counted apart, in one row and alone; few values, many times."""
    V = 20011
    l, u = inputs(16, V, "bf16", seed=8)
    f = l.float()
    f[0] *= 2.0 ** -12
    f[1] *= 2.0 ** 12
    f[2, ::2] *= 2.0 ** -10
    f[3, ::2] *= 2.0 ** 7
    f[4] = f[4].abs() + 250
    f[5] = 256 - f[5].abs() * 2
    f[6] = 2.0 ** -8
    f[7] = -2.0 ** -8
    f[7, ::3] = 2.0 ** -9
    f[8] = -3e38
    f[8, 5::1000] = -2.9e38
    f[9] = f[9].round()
    f[10, ::2] = -INF
    f[11, 1::2] = float("nan")
    f[12, 77] = INF
    f[13] = 0.0
    f[13, ::2] = -0.0
    f[14] = (f[14] * 4).round() / 4 + 255
    l = f.bfloat16()
    for kw in FILTERS:
        check(l, u, **kw)
    for T in (100.0, 1e-3):
        check(l, u, T=T, p=0.9)
        check(l, u, T=T, k=300, p=0.9)
