"""I8Linear and the integer experts with rows next to the ends of fp32's range: a product of the two scales alone would
leave it where the output does not.  Tolerance as in test_gpu_i8_linear.py: 6 roundings of 2^-24 of the terms, half a step of
bf16."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_i8_linear import U, layer, quantised  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,K,M", [(3, 256, 64), (40, 256, 37), (700, 512, 1024), (3000, 512, 2051)])
def test_scales_whose_product_leaves_the_range(N, K, M, act):
    gen = torch.Generator(device="cuda").manual_seed(N)
    x = torch.randn(N, K, generator=gen, device="cuda")
    x = x / x.abs().amax(1, keepdim=True)
    x[0::3] *= 1e38          # a sum of 0: 0 (or the bias), whatever the scales
    x[1::3] *= 1e-28         # scales of 8e-31 and 1e-9, whose product has 19 bits, and sums of 5e4: outputs of 4e-35
    x[0::3, K // 2:] = x[0::3, :K // 2]
    x = x.to(torch.float32 if act == "f32" else torch.bfloat16)
    w = torch.randint(-127, 128, (M, K), generator=gen, device="cuda", dtype=torch.int8)
    w[:, K // 2:] = -w[:, :K // 2]
    s = torch.rand(M, generator=gen, device="cuda") + 0.5
    big, small = s * 1e4, s * 1e-9
    b = torch.randn(M, generator=gen, device="cuda")
    y = layer(K, M, act, w, big, b).forward(x)[0::3]
    assert torch.equal(y, b.to(y.dtype).expand_as(y))
    w = torch.randint(-127, 128, (M, K), generator=gen, device="cuda", dtype=torch.int8)
    y = layer(K, M, act, w, small, None).forward(x)[1::3]
    q, sx = quantised(x[1::3])
    acc = q @ w.double().t()
    want = acc * sx[:, None] * small.double()
    # (of terms that are numbers of full precision: 2^-126 and up)
    normal = want.abs() > 2.0 ** -120
    assert normal.float().mean() > 0.5
    half = U if act == "f32" else 2.0 ** -8
    assert ((y.double() - want).abs() <= (6 * U + half) * want.abs())[normal].all()
