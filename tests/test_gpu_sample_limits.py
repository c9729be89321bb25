"""Sampler: min_p down to the units of the weights.  The reference and its tolerances are test_gpu_sample.py's."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_sample import check  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("V", [600, 8000, 30000])
@pytest.mark.parametrize("units", [1, 2, 3, 11, 70])
def test_min_p_of_a_few_units(V, units):
    """A weight that rounds up to min_p's units is kept: logits around the half unit below, and u where they count."""
    gen = torch.Generator(device="cuda").manual_seed(V + units)
    # (2^40 exp(l) between units - 0.9 and units + 0.4, none within 0.001 of a half, where the exponential's own rounding
    # decides; all but one of a row)
    f = torch.rand(6, V, generator=gen, device="cuda", dtype=torch.float64) * 1.3 - 0.9
    f = torch.where((f + 0.5).abs() < 0.001, f + 0.01, f)
    l = (((units + f) * 2.0 ** -40).log()).float()
    l[:, V // 3] = 0.0
    # what lies before the largest logit, by id, is drawn by a u this small, what lies behind it by one near 1
    u = torch.tensor([0.0, 2.0 ** -42, 2.0 ** -36, 1 - 2.0 ** -24, 0.5, 1e-12], device="cuda")
    for m in (units * 2.0 ** -40, (units - 0.4) * 2.0 ** -40):
        for kw in (dict(), dict(p=0.9999999), dict(k=100), dict(k=V // 2), dict(k=200, p=1 - 2.0 ** -24)):
            check(l, u, m=m, **kw)
    token, kept = check(l, u, m=units * 2.0 ** -40)
    assert (token != V // 3).any()
