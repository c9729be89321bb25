"""MoELayer(weights="i8") held to its formula as tightly as the caller's type allows.

fp32 callers: hidden units are numbers of 32 bits, each operation rounded by itself, and scales max (1 / 127), both of 32
bits, as a torch program has them on the GPU: their integers are that program's, every one.  What follows is smooth: per
output, the sum as a float, its two products, the bias, the weight and the sums over the token's experts round once each,
6 + k steps of 2^-24 of the terms' magnitudes.  A unit on the other side of a border would be a step, max|h| / 127 times a
weight, thousands of times as much.

bf16 callers: outputs of an expert keep 2^-16 of themselves, whatever the other channels' sizes; y is rounded to bf16 (2^-8).
What hidden units of 20 bits do to a channel is a sum of integer steps, which the channel's own weights scale.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_i8_experts import Layer  # noqa: E402

U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def rows8(a):
    """(integers in 64 bits, scales in 32) of rows of 32 bits."""
    top = a.abs().amax(-1, keepdim=True)
    q = (a.double() * (127 * (1 / top.double().clamp(min=1e-300)))).round()
    return q, (top * torch.tensor(1 / 127, dtype=torch.float32, device=a.device)).squeeze(-1)


def program(L, x, idx, w):
    """(y, the terms' magnitudes) in 64 bits, but for the hidden units."""
    y = torch.zeros(x.shape[0], L.C, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(y)
    for e in range(L.E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        W = {n: rows8(L.W[n][e].t().contiguous()) for n in "gud"}

        def product(a, n):
            q, sa = rows8(a)
            acc = q @ W[n][0].t()
            return acc, sa, W[n][1]

        def floats(acc, sa, sw, b):
            assert acc.abs().max() < 2 ** 24
            return acc.float() * sa[:, None] * sw + b

        g, u = (floats(*product(x[t], n), L.b[n][e]) for n in "gu")
        h = g / (1 + (-g).exp()) * u
        acc, sa, sw = product(h, "d")
        o = acc * sa.double()[:, None] * sw.double()
        p = w[t, j].double()[:, None]
        y.index_add_(0, t, (o + L.b["d"][e].double()) * p)
        mag.index_add_(0, t, (o.abs() + L.b["d"][e].double().abs()) * p.abs())
    return y, mag


@pytest.mark.parametrize("N,C,H,E,k", [(1, 64, 96, 4, 2), (64, 1024, 704, 64, 8), (33, 100, 77, 5, 3), (1024, 512, 1024, 8, 2),
                                       (2048, 1024, 2816, 8, 2), (12541, 240, 608, 16, 3), (16384, 512, 1376, 8, 2),
                                       (3000, 256, 512, 96, 8)])
def test_integers_of_fp32_callers(N, C, H, E, k):
    L = Layer(C, H, E, k, "f32", seed=N)
    for seed in (2, 3):
        x, idx, w = L.inputs(N, seed)
        y = L.op.forward_routed(x, idx, w)
        want, mag = program(L, x, idx, w)
        bad = ((y.double() - want).abs() > (6 + k) * U * mag).any(1)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].flatten().tolist())
        assert ((y.double() - want).norm() / want.norm()).item() < 2e-6


def big_channels(L, at, factor):
    """The same layer, the output channels `at` factor times as large."""
    params = [L.wr, L.br]
    L.W["d"][:, :, at] *= factor
    L.b["d"][:, at] *= factor
    for e in range(L.E):
        for n in "gud":
            params += [L.W[n][e], L.b[n][e]]
    L.op.load_parameters(params)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("N", [40, 600])
@pytest.mark.parametrize("factor", [1.0, 256.0, 4096.0, 32768.0])
def test_channels_of_other_sizes(factor, N, act):
    L = Layer(256, 384, 4, 2, act)
    big_channels(L, slice(5, None, 32), factor)
    x, idx, w = L.inputs(N)
    y = L.op.forward_routed(x, idx, w)
    want = L.check(y, x, idx, w)     # each output, by its own terms
    # each channel: y's rounding, 2^-8 of each, and the integer steps: with a probability of 1 / 6000 (2^-22 for fp32)
    # for each of 384 units of 2 experts, a step is 1 / (sqrt(384) 20) of an output and of 40 rows 8 have one: 0.0012; twice that
    off = (y.double() - want).norm(dim=0) / want.norm(dim=0)
    assert off.max().item() < (2.0 ** -8 + 0.0024 if act == "bf16" else 0.0006), off.max().item()


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_an_infinite_channel_leaves_the_others(act):
    L = Layer(128, 256, 4, 2, act)
    x, idx, w = L.inputs(50)
    clean = L.op.forward_routed(x, idx, w)
    L.b["d"][:, 37] = float("inf")
    L.b["d"][:, 70] = float("nan")
    big_channels(L, slice(0, 0), 1.0)
    y = L.op.forward_routed(x, idx, w)
    keep = [c for c in range(128) if c not in (37, 70)]
    assert torch.equal(y[:, keep], clean[:, keep])
    assert (y[:, 37] == float("inf")).all() and y[:, 70].isnan().all()
