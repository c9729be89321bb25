"""The loss' gradients for upstream gradients of any size: relative errors as for ones
near 1, by test_gpu_lm_loss's tolerances, here with no more slack than the smallest
number of the outputs' type."""
import pytest

from test_gpu_lm_loss import inputs, reference, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-37, 1e-35, 1e-31, 1e-20, 1e20, 1e31, 1e36])
def test_upstream_gradients_of_any_size(act, size):
    x, W, b, t = inputs(300, 256, 500, act)
    t[::7] = -1
    g = size * torch.randn(300, generator=torch.Generator().manual_seed(5)).clamp(-2, 2).cuda()
    got, ref = run(x, W, b, t, act, dloss=g), reference(x, W, b, t, g)
    for k in ("dx", "dW", "db"):
        want, tol = ref[k]
        least = 2.0 ** -149 if act == "f32" or k == "db" else 2.0 ** -133
        err = (got[k].double() - want).abs()
        assert (err <= tol + 2 * least).all(), (k, float((err / (tol + 2 * least)).max()))
