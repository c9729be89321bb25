"""The training step's operators on tensors whose byte offsets pass 32 bits:
the far end against 64 bits, by the tolerances of the small cases."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def test_loss_over_a_vocabulary_past_4_gib():
    from mgpt_amd.loss import LMLoss
    N, C, V = 70, 8192, 300001
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(N, C, generator=gen, device="cuda").bfloat16()
    W = torch.empty(V, C, dtype=torch.bfloat16, device="cuda")
    for r in range(0, V, 50000):
        W[r:r + 50000] = torch.randn(min(50000, V - r), C, generator=gen, device="cuda") * 0.01
    t = torch.randint(0, V, (N,), generator=gen, device="cuda", dtype=torch.int32)
    t[0], t[1], t[2] = V - 1, 0, -1
    op = LMLoss(C, V)
    loss, lse, mean = op.forward(x, W, t)
    dx, dW, _ = op.backward(x, W, t, lse)
    xd = x.double()
    z = torch.cat([xd @ W[r:r + 50000].double().t() for r in range(0, V, 50000)], 1)
    ref = torch.logsumexp(z, 1)
    # (C + 2) u of a logit's terms, about 0.01 sqrt(2 / pi) |x| C in sum, and a few hundred
    # roundings of a log-sum-exp near 13
    tol = (C + 2) * U * 0.008 * float(xd.abs().sum(1).max()) + 300 * U * 13
    assert float((lse.double() - ref).abs().max()) <= tol
    has = t >= 0
    d = (z - ref[:, None]).exp()
    d[has, t[has].long()] -= 1
    d[~has] = 0
    d /= int(has.sum())
    for rows in (slice(0, 300), slice(V - 300, V)):
        want = d[:, rows].t() @ xd
        amp = d[:, rows].abs().t() @ xd.abs()
        # d and the result round to bf16 (2^-8 of each at most)
        assert (dW[rows].double() - want).abs().le(2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * tol + N * U) * amp).all()
    want = sum(d[:, r:r + 50000] @ W[r:r + 50000].double() for r in range(0, V, 50000))
    err = float((dx.double() - want).norm() / want.norm())
    assert err <= 2.0 ** -7
    assert not dx[2].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_past_4_gib(bits):
    from mgpt_amd.optim import AdamW
    n = (1 << 30) + 4097 * 256 + 5
    p = torch.zeros(n, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(70000, generator=torch.Generator().manual_seed(3))
    p[-70000:] = tail.cuda()
    g[-70000:] = tail.flip(0).cuda().bfloat16()
    first = p[:1000].clone()
    opt = AdamW([p], lr=1e-2, state_bits=bits)
    opt.step([g])
    q, h = p[-70000:].double().cpu().numpy(), g[-70000:].double().cpu().numpy()
    m, v = 0.1 * h, 0.001 * h * h
    want = tail.double().numpy() * (1 - 1e-4) - 1e-2 * (m / 0.1) / (np.sqrt(v / 0.001) + 1e-8)
    # betas, lr and weight_decay are held in fp32: each off by at most u of itself; the
    # second moment's correction 1 / (1 - b2) by u / 0.001
    assert np.abs(q - want).max() <= 1e-2 * 2 * U / 0.001 + 8 * U * 5
    assert torch.equal(p[:1000], first)
    assert not opt.m[:1000].float().any()


def test_norms_past_4_gib():
    from mgpt_amd.norm import ResidualNorm
    N, C = 280001, 8192
    op = ResidualNorm(C, act="bf16")
    x = torch.zeros(N, C, dtype=torch.bfloat16, device="cuda")
    h = torch.zeros_like(x)
    gen = torch.Generator(device="cuda").manual_seed(5)
    x[-40:] = torch.randn(40, C, generator=gen, device="cuda").bfloat16()
    h[-40:] = torch.randn(40, C, generator=gen, device="cuda").bfloat16()
    kw = dict(gamma_post=torch.full((C,), 0.5, device="cuda"), gate=torch.full((C,), 2.0, device="cuda"),
              gamma_pre=torch.full((C,), 3.0, device="cuda"))
    out, y, rh, ro = op.forward(x, h, **kw)
    dx, dh, dpost, dgate, dpre = op.backward(x, h, None, x, rh, ro, **kw)
    xs, hs, last = x[-40:].contiguous(), h[-40:].contiguous(), slice(N - 40, N)
    o2, y2, rh2, ro2 = op.forward(xs, hs, **kw)
    dx2, dh2, dpost2, dgate2, dpre2 = op.backward(xs, hs, None, xs, rh2, ro2, **kw)
    for a, b in ((out, o2), (y, y2), (rh, rh2), (ro, ro2), (dx, dx2), (dh, dh2)):
        assert torch.equal(a[last], b)
        assert not a[:64].any() or a is rh or a is ro
    # the other rows add zeros to the column sums, in another order of the 40
    for a, b in ((dpost, dpost2), (dgate, dgate2), (dpre, dpre2)):
        assert float((a - b).norm() / b.norm()) <= 64 * U
