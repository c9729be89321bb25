"""MoELayer(weights="i8") held to its formula as tightly as the caller's type allows.

fp32 callers: hidden units are numbers of 32 bits, each operation rounded by itself, and scales max (1 / 127), both of 32
bits, as a torch program has them on the GPU: their integers are that program's, every one.  What follows is smooth: per
output, the sum as a float, its two products, the bias, the weight and the sums over the token's experts round once each,
6 + k steps of 2^-24 of the terms' magnitudes.  A unit on the other side of a border would be a step, max|h| / 127 times a
weight, thousands of times as much.
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
