"""I8Linear (mgpt_i8_*) against its formula: the integers exactly, the rest in 64 bits.

Tolerance, u = 2^-24: the sum as a float, the token's scale, its product with the output's,
the product and the bias each round once: 6 u of the terms' magnitudes, and half a step of the
output's type, 2^-8 of the value in bf16.  The integers are the same on both sides: x times 127 (1 / max|x|), in 64 bits.
"""
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


def quantised(x):
    top = x.double().abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(x.double() * (127 / top)), torch.zeros(()).double().to(x.device))
    return q, (top / 127).squeeze(1)


def inputs(N, K, M, act, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, K, generator=gen, device="cuda") * torch.exp(torch.randn(N, 1, generator=gen, device="cuda"))
    x = x.to(torch.float32 if act == "f32" else torch.bfloat16)
    w = torch.randint(-127, 128, (M, K), generator=gen, device="cuda", dtype=torch.int8)
    s = torch.rand(M, generator=gen, device="cuda") + 0.01
    b = torch.randn(M, generator=gen, device="cuda") * 10
    return x, w, s, b


def check(op, x, w, s, b):
    y = op.forward(x)
    q, sx = quantised(x)
    acc = q @ w.double().t()
    want = acc * sx[:, None] * s.double()
    mag = want.abs()
    if b is not None:
        want, mag = want + b.double(), mag + b.double().abs()
    half = U if x.dtype == torch.float32 else 2.0 ** -8
    assert y.dtype == x.dtype and y.shape == (x.shape[0], w.shape[0])
    bad = (y.double() - want).abs() > 6 * U * mag + half * want.abs() + 1e-37
    assert not bad.any(), (bad.nonzero()[:5], y[bad][:5], want[bad][:5])
    assert torch.equal(y, op.forward(x))


def layer(K, M, act, w, s, b):
    from mgpt_amd.linear8 import I8Linear
    op = I8Linear(K, M, act=act)
    op.load_quantized(w, s, bias=b)
    return op


# few rows (the stream kernel: contractions split 1 to 8 times, one and two row blocks), 128 x 128 and 256 x 256 tiles,
# odd sizes, one of each
SHAPES = [(1, 1, 1), (1, 128, 32), (1, 2048, 5003), (2, 100, 8), (5, 4096, 264), (31, 129, 40), (32, 640, 1000),
          (33, 300, 72), (64, 1024, 4096), (50, 2048, 9), (64, 16384, 100), (65, 127, 128), (100, 512, 1003), (129, 1000, 136),
          (257, 384, 520), (999, 500, 1003), (300, 4100, 777), (2048, 256, 8192), (4097, 1024, 4100), (8192, 130, 2048),
          (5000, 640, 3333)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,K,M", SHAPES)
def test_shapes(N, K, M, act):
    x, w, s, b = inputs(N, K, M, act, seed=N + K + M)
    check(layer(K, M, act, w, s, b), x, w, s, b)
    check(layer(K, M, act, w, s, None), x, w, s, None)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_float_weights(act):
    """Rows of a float weight, quantised by the layer as a token's are."""
    from mgpt_amd.linear8 import I8Linear
    gen = torch.Generator(device="cuda").manual_seed(4)
    for M, K, dt in ((1000, 333, torch.float32), (64, 2048, torch.bfloat16), (33, 5000, torch.float32)):
        W = (torch.randn(M, K, generator=gen, device="cuda") * torch.rand(M, 1, generator=gen, device="cuda")).to(dt)
        W[5] = 0
        op = I8Linear(K, M, act=act)
        op.load(W)
        q, s = quantised(W)
        assert ((op.scales.double() - s).abs() <= U * s).all()
        for N in (3, 200):
            x = inputs(N, K, 1, act)[0]
            check(op, x, q.to(torch.int8), op.scales, None)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_rows_of_any_size(act):
    """Rows of zeros, of the smallest and the largest numbers, ties between integers; rows that are not finite."""
    for N, K, M in ((40, 200, 64), (300, 200, 24), (300, 1000, 4096)):
        x, w, s, b = inputs(N, K, M, act)
        x[0] = 0
        x[1] = -0.0
        x[2] = 0
        x[2, 7] = 1e-45 if act == "f32" else 1e-40
        x[3] = torch.finfo(x.dtype).tiny
        x[4] *= 1e-30
        x[5] = torch.arange(K, device="cuda") % 255 - 127
        x[6] = (torch.arange(K, device="cuda") % 509 - 254) * 0.5       # ties
        x[7] *= 1e30
        s = s * 1e-5
        b = b * 0
        op = layer(K, M, act, w, s, b)
        check(op, x, w, s, b)
        clean = op.forward(x)
        for bad in (float("nan"), float("inf"), -float("inf")):
            z = x.clone()
            z[9, K - 1] = bad
            z[20, 0] = bad
            y = op.forward(z)
            assert y[9].isnan().all() and y[20].isnan().all()
            keep = [i for i in range(N) if i not in (9, 20)]
            assert torch.equal(y[keep], clean[keep])


def test_the_longest_contraction():
    """2^17 products of 127 by 127 fit the integers."""
    K = 1 << 17
    for N in (1, 70):
        x = torch.ones(N, K, device="cuda")
        x[0, 1::2] = -1
        w = torch.full((40, K), 127, dtype=torch.int8, device="cuda")
        w[1] = -127
        s = torch.ones(40, device="cuda")
        y = layer(K, 40, "f32", w, s, None).forward(x)
        want = torch.full((N, 40), 127.0 * K, device="cuda")
        want[:, 1] *= -1
        want[0] = 0
        assert ((y - want).abs() <= 6 * U * want.abs()).all()


def test_rows_at_any_element_other_streams_graphs():
    K, M = 136, 200
    x, w, s, b = inputs(90, K, M, "bf16")
    op = layer(K, M, "bf16", w, s, b)
    want = op.forward(x)
    flat = torch.empty(90 * K + 8, dtype=torch.bfloat16, device="cuda")
    for off in (0, 1, 2, 5):
        v = flat[off:off + 90 * K].view(90, K)
        v.copy_(x)
        assert torch.equal(op.forward(v), want)
    assert torch.equal(op.forward(x.view(3, 30, K)).view(90, M), want)
    assert op.forward(x[:0]).shape == (0, M)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = op.forward(x)
    st.synchronize()
    assert torch.equal(got, want)
    for n in (4, 90):
        buf = x[:n].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = op.forward(buf)
        for seed in (2, 3, 4):
            buf.copy_(inputs(n, K, M, "bf16", seed)[0])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, op.forward(buf))


def test_offsets_past_32_bits():
    """Outputs past 2^32 bytes, a weight past 2^31."""
    N, K, M = 70000, 64, 32768
    x, w, s, b = inputs(N, K, M, "bf16")
    y = layer(K, M, "bf16", w, s, b).forward(x)
    op = layer(K, M, "bf16", w, s, b)
    assert torch.equal(y[-40:], op.forward(x[-40:].contiguous()))
    del y
    K, M = 16384, 140000
    w = torch.randint(-127, 128, (M, K), device="cuda", dtype=torch.int8)
    s = torch.rand(M, device="cuda")
    x = inputs(300, K, 1, "bf16")[0]
    op = layer(K, M, "bf16", w, s, None)
    tail = layer(K, 256, "bf16", w[-256:].contiguous(), s[-256:].contiguous(), None)
    for n in (3, 300):
        assert torch.equal(op.forward(x[:n].contiguous())[:, -256:], tail.forward(x[:n].contiguous()))
