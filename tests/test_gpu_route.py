"""mgpt_route_forward / _backward / _balance against the formulas in 64 bits.

The chosen experts have to be equal.  Tolerances, u = 2^-24: a score is within
(16 + V + 2 |x|) u of itself, x the exponent's argument (under 40 here), V <= 14 additions of a row's sum; the weights'
sum adds 8, the quotients 4: 128 u.  A gradient is a sum of products of such: 512 u of its terms'
magnitudes, and half a step of its type, 2^-8 of it in bf16.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
INF = float("inf")
BIG = torch.finfo(torch.float32).max


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def scores(l, score):
    l = torch.where(l.isnan(), torch.full_like(l, -INF), l.clamp(max=BIG))
    if score == "sigmoid":
        return l, torch.sigmoid(l)
    top = l.amax(1, keepdim=True)
    z = (l - torch.where(top > -INF, top, torch.zeros_like(top))).exp()
    total = z.sum(1, keepdim=True)
    return l, torch.where(total > 0, z / total, torch.zeros_like(z))


def reference(logits, bias, k, score, groups, top_groups, group_best, renormalise, scale):
    """(idx, weights, scores) row by row in 64 bits on the CPU."""
    l, s = scores(logits.double().cpu(), score)
    N, E = l.shape
    size = s if bias is None else s + bias.double().cpu()
    size = torch.where((l > -INF) & ~size.isnan(), size, torch.full_like(s, -INF))
    key = torch.where(size > -INF, l if bias is None else size, size)
    if groups > 1:
        best = size.view(N, groups, -1).sort(dim=2, descending=True)[0][:, :, :group_best]
        total = torch.where(best > -INF, best, torch.zeros_like(best)).sum(2)
        total = torch.where(best[:, :, 0] > -INF, total, torch.full_like(total, -INF))
        order = total.sort(dim=1, descending=True, stable=True)[1][:, :top_groups]
        on = torch.zeros(N, groups, dtype=torch.bool).scatter_(1, order, True)
        key = torch.where(on.repeat_interleave(E // groups, 1), key, torch.full_like(key, -INF))
    top, idx = key.sort(dim=1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k]
    sel = torch.where(top > -INF, s.gather(1, idx), torch.zeros(()).double())
    w = sel * scale
    if renormalise:
        w = w / (sel.sum(1, keepdim=True) + 1e-20)
    return idx, w, top > -INF


def gradient(logits, idx, on, dw, dscores, score, renormalise, scale):
    """(dl, the magnitude of its terms) in 64 bits."""
    l, s = scores(logits.double().cpu(), score)
    dw = torch.where(on, dw.double().cpu(), torch.zeros(()).double())
    sel = torch.where(on, s.gather(1, idx), torch.zeros(()).double())
    d, a = scale * dw, abs(scale) * dw.abs()
    if renormalise:
        D = sel.sum(1, keepdim=True) + 1e-20
        d = (d - (d * sel).sum(1, keepdim=True) / D) / D
        a = (a + (a * sel).sum(1, keepdim=True) / D) / D
    d, a = (torch.where(on, x, torch.zeros(()).double()) for x in (d, a))
    ds = torch.zeros_like(s).scatter_add_(1, idx, d)
    da = torch.zeros_like(s).scatter_add_(1, idx, a)
    if dscores is not None:
        ds, da = ds + dscores.double().cpu(), da + dscores.double().cpu().abs()
    if score == "sigmoid":
        t = s * torch.sigmoid(-l)
        dl, am = ds * t, da * t
    else:
        dl = s * (ds - (ds * s).sum(1, keepdim=True))
        am = s * (da + (da * s).sum(1, keepdim=True))
    off = ~(l > -INF)
    return dl.masked_fill(off, 0), am.masked_fill(off, 0)


def check(logits, k, score="softmax", bias=None, groups=1, top_groups=None, group_best=2, renormalise=True, scale=1.0,
          dscores=None, seed=3):
    from mgpt_amd.routing import ExpertRouting
    N, E = logits.shape
    act = "f32" if logits.dtype == torch.float32 else "bf16"
    op = ExpertRouting(E, k, score=score, groups=groups, top_groups=top_groups, group_best=group_best,
                       renormalise=renormalise, scale=scale, act=act)
    counts = torch.full((E,), 5, dtype=torch.int32, device="cuda")
    idx, w = op.forward(logits, bias=bias, counts=counts)
    ri, rw, on = reference(logits, bias, k, score, groups, op.config.top_groups, group_best, renormalise, scale)
    assert torch.equal(idx.cpu().long(), ri)
    assert ((w.double().cpu() - rw).abs() <= 128 * U * rw.abs() + 1e-37).all()
    assert (w.cpu()[~on] == 0).all()
    assert torch.equal(counts.cpu().long() - 5, torch.bincount(ri[on], minlength=E))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dw = torch.randn(N, k, generator=gen, device="cuda")
    dl = op.backward(logits, idx, w, dw, dscores=dscores)
    assert dl.dtype == logits.dtype
    rd, mag = gradient(logits, ri, on & (rw.float() != 0), dw, dscores, score, renormalise, scale)
    half = 2.0 ** -8 if act == "bf16" else U
    assert ((dl.double().cpu() - rd).abs() <= 512 * U * mag + half * rd.abs() + 1e-37).all()
    # the same call gives the same bits
    assert torch.equal(idx, op.forward(logits, bias=bias)[0])
    assert torch.equal(dl, op.backward(logits, idx, w, dw, dscores=dscores))
    return idx, w, dl


def logits_of(N, E, act, seed=1, std=1.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    l = torch.randn(N, E, generator=gen, device="cuda") * std
    return l.to(torch.float32 if act == "f32" else torch.bfloat16)


def bias_of(E, seed=2, std=0.05):
    return torch.randn(E, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * std


SHAPES = [(1, 1, 1), (1, 2, 2), (3, 5, 5), (65, 8, 2), (257, 16, 2), (130, 17, 3), (64, 32, 8), (77, 33, 4), (64, 64, 8),
          (1000, 60, 6), (33, 128, 8), (129, 127, 7), (50, 160, 6), (300, 256, 8), (41, 257, 8), (37, 511, 5), (19, 512, 8)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,E,k", SHAPES)
def test_shapes(N, E, k, act):
    l = logits_of(N, E, act, seed=N + E)
    check(l, k)
    check(l, k, "sigmoid", bias_of(E), renormalise=True, scale=2.5, dscores=bias_of(E, 4, 0.1))
    check(l, k, "softmax", bias_of(E), renormalise=False, dscores=bias_of(E, 5, 0.1))
    check(l, k, "sigmoid", renormalise=False, scale=0.5)


@pytest.mark.parametrize("E,groups,top_groups", [(8, 2, 1), (12, 4, 2), (16, 16, 3), (64, 8, 4), (60, 6, 2), (160, 8, 3),
                                                 (256, 8, 4), (255, 5, 2), (512, 64, 20), (384, 3, 1), (64, 64, 9),
                                                 (130, 65 - 52, 4)])
@pytest.mark.parametrize("best", [1, 2])
def test_groups(E, groups, top_groups, best):
    k = min(8, E // groups * top_groups)
    for act in ("f32", "bf16"):
        l = logits_of(203, E, act, seed=E)
        for score in ("softmax", "sigmoid"):
            for b in (None, bias_of(E)):
                check(l, k, score, b, groups, top_groups, best)


def test_fewer_than_k_take_part():
    """Groups and masks that leave fewer experts than k: the lowest other ids, weight 0."""
    check(logits_of(70, 16, "f32"), 8, "softmax", None, 8, 2, 1)
    check(logits_of(70, 16, "f32"), 8, "sigmoid", bias_of(16), 8, 3, 2)
    for E in (16, 48, 200):
        l = logits_of(90, E, "f32")
        l[::2, 5:] = -INF
        l[1::3, :E - 2] = -INF
        l[7] = -INF
        l[8] = float("nan")
        l[9, ::2] = float("nan")
        l[10, 3] = INF
        l[11, 4:6] = INF
        l[12] = INF
        l[13] = -BIG
        l[14, 1] = BIG
        b = bias_of(E)
        b[2] = -INF
        for score in ("softmax", "sigmoid"):
            check(l, 8, score)
            check(l, 8, score, b)
            check(l, 8, score, None, 4, 2)
            check(l, 8, score, b, 4, 3, dscores=bias_of(E, 6))
        b[3] = float("nan")
        b[4] = INF
        check(l, 8, "sigmoid", b, renormalise=False)


@pytest.mark.parametrize("E,groups", [(16, 1), (64, 4), (256, 8), (500, 5)])
def test_ties(E, groups):
    """Equal keys: the lower id first, also where the bias makes the keys equal."""
    gen = torch.Generator(device="cuda").manual_seed(E)
    l = torch.randint(-1, 2, (150, E), generator=gen, device="cuda").float()
    l[0] = 0
    for score in ("softmax", "sigmoid"):
        check(l, 8, score, None, groups, max(1, groups // 2))
        check(l, 8, score, torch.zeros(E, device="cuda"), groups, max(1, groups // 2))
        check(l, 8, score, torch.randint(0, 3, (E,), generator=gen, device="cuda") * 0.25, groups, max(1, groups // 2))


@pytest.mark.parametrize("E", [16, 64, 256])
def test_keys_that_fp32_cannot_tell_apart(E):
    """A bias that cancels the scores' differences up to some 2^-26: 64 bits decide."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    base = torch.randn(E, generator=gen, device="cuda")
    b = (1.0 - torch.sigmoid(base.double())).float()
    l = base + torch.randn(400, E, generator=gen, device="cuda") * 2.0 ** -22
    check(l, 8, "sigmoid", b)
    check(l, 8, "sigmoid", b, 4, 2)


def test_far_logits():
    l = logits_of(100, 64, "f32", std=30.0)
    from mgpt_amd.routing import ExpertRouting
    for score in ("softmax", "sigmoid"):
        op = ExpertRouting(64, 8, score=score)
        idx, w = op.forward(l)
        ri, rw, _ = reference(l, None, 8, score, 1, 1, 2, True, 1.0)
        assert torch.equal(idx.cpu().long(), ri)
        assert ((w.double().cpu() - rw).abs() <= 1024 * U * rw.abs() + 1e-30).all()   # (|x| up to 250)


def test_gradient_against_differences():
    """Central differences of sum(w dw) in 64 bits, the choice held."""
    l = logits_of(6, 24, "f32")
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            idx, w, dl = check(l, 4, score, None, 1, 1, 2, renorm, 1.5, seed=11)
            dw = torch.randn(6, 4, generator=torch.Generator(device="cuda").manual_seed(11), device="cuda").double().cpu()

            def f(x):
                s = scores(x, score)[1].gather(1, idx.cpu().long())
                s = s * 1.5
                return ((s / (s.sum(1, keepdim=True) / 1.5 + 1e-20) if renorm else s) * dw).sum()

            x = l.double().cpu()
            for e in range(24):
                h = torch.zeros_like(x)
                h[3, e] = 1e-5
                assert abs((f(x + h) - f(x - h)) / 2e-5 - dl[3, e].item()) < 1e-6


def test_rows_at_any_element_and_other_devices_streams():
    from mgpt_amd.routing import ExpertRouting
    flat = logits_of(1, 40 * 64 + 3, "f32").view(-1)
    for off in (0, 1, 2, 3):
        check(flat[off:off + 40 * 64].view(40, 64), 6, "sigmoid", bias_of(64))
    op = ExpertRouting(64, 6)
    l = logits_of(512, 64, "f32")
    want = op.forward(l)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = op.forward(l)
    st.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    # leading dimensions, and no tokens
    a = op.forward(l.view(2, 4, 64, 64))
    assert a[0].shape == (2, 4, 64, 6) and torch.equal(a[0].view(-1, 6), want[0])
    e = op.forward(l[:0])
    assert e[0].shape == (0, 6) and op.backward(l[:0], *e, e[1]).shape == (0, 64)


def test_offsets_past_32_bits():
    from mgpt_amd.routing import ExpertRouting
    N, E = (1 << 22) + 37, 512
    l = torch.zeros(N, E, dtype=torch.bfloat16, device="cuda")
    tail = logits_of(64, E, "bf16")
    l[-64:] = tail
    op = ExpertRouting(E, 8, act="bf16")
    idx, w = op.forward(l)
    ri, rw, _ = reference(tail, None, 8, "softmax", 1, 1, 2, True, 1.0)
    assert torch.equal(idx[-64:].cpu().long(), ri)
    assert torch.equal(idx[0].cpu(), torch.arange(8, dtype=torch.int32))
    dl = op.backward(l, idx, w, torch.ones_like(w))
    want = op.backward(tail, idx[-64:].contiguous(), w[-64:].contiguous(), torch.ones(64, 8, device="cuda"))
    assert torch.equal(dl[-64:], want)


def test_replayed_graph():
    from mgpt_amd.routing import ExpertRouting
    op = ExpertRouting(64, 8, score="sigmoid", groups=8, top_groups=4)
    l, b = logits_of(300, 64, "f32"), bias_of(64)
    counts = torch.zeros(64, dtype=torch.int32, device="cuda")
    dw = torch.randn(300, 8, device="cuda")
    op.forward(l, b, counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        counts.zero_()
        idx, w = op.forward(l, b, counts)
        dl = op.backward(l, idx, w, dw)
        op.balance(b, counts, 0.01)
    for seed in (5, 6, 7):
        l.copy_(logits_of(300, 64, "f32", seed))
        before = b.clone()
        graph.replay()
        torch.cuda.synchronize()
        ei, ew = op.forward(l, before)
        assert torch.equal(idx, ei) and torch.equal(w, ew) and torch.equal(dl, op.backward(l, ei, ew, dw))
        c = torch.bincount(ei.view(-1).long(), minlength=64)
        assert torch.equal(counts.long(), c)
        want = before + 0.01 * torch.sign(c.double().mean() - c.double()).float()
        assert torch.equal(b, want)


def test_balance_evens_the_load():
    from mgpt_amd.routing import ExpertRouting
    op = ExpertRouting(32, 4, score="sigmoid")
    l = logits_of(4096, 32, "f32") + torch.linspace(-1, 1, 32, device="cuda")
    b = torch.zeros(32, device="cuda")

    def load():
        c = torch.zeros(32, dtype=torch.int32, device="cuda")
        op.forward(l, b, c)
        return c

    first = load()
    for _ in range(200):
        op.balance(b, load(), 0.005)
    last = load()
    assert int(first.sum()) == int(last.sum()) == 4096 * 4
    assert int(last.max()) - int(last.min()) < (int(first.max()) - int(first.min())) // 4


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("E,groups", [(3, 1), (16, 4), (60, 1), (160, 8), (256, 8), (512, 1)])
def test_far_logits_beside_masked_ones(E, groups, act):
    """Experts that are out come behind all that are not, however far those lie below the largest."""
    N = 200
    gen = torch.Generator(device="cuda").manual_seed(E)
    for gap in (20.0, 31.0, 34.0, 60.0, 300.0, 1e5):
        l = logits_of(N, E, act, seed=E)
        l[:, ::2] = -INF
        l[:, 1::4] -= gap
        l[torch.arange(N, device="cuda"), torch.randint(0, E, (N,), generator=gen, device="cuda")] = 3.0
        l[5] = -INF
        l[5, E - 1] = -gap
        for k in (1, min(4, E), min(8, E)):
            for score in ("softmax", "sigmoid"):
                check(l, k, score, renormalise=False)
                if groups > 1:
                    check(l, k, score, groups=groups, top_groups=max(1, groups // 2), renormalise=False)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_of_the_smallest_scores(score):
    """Sizes of groups down to 64 bits' smallest normal number are in order."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    l = -694 - 13 * torch.rand(300, 16, generator=gen, device="cuda")
    if score == "softmax":
        l[:, 0] = 0.0
    for groups, top in ((16, 5), (8, 3), (4, 2)):
        check(l, 2, score, groups=groups, top_groups=top, renormalise=False)
