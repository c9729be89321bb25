"""Sampler: min_p down to the units of the weights, parameters that are no numbers, very many rows.
The reference and its tolerances are test_gpu_sample.py's."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_sample import check, inputs  # noqa: E402


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


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("V", [500, 8000, 9001, 30000])
def test_parameters_that_are_no_numbers(V, act):
    """NaN in a device array: temperature and u as 0, top_p and min_p as no restriction."""
    from mgpt_amd.sampling import Sampler
    B = 12
    l, u = inputs(B, V, act, seed=V)
    op = Sampler(V, act=act)
    full = lambda v: torch.full((B,), v, device="cuda")  # noqa: E731
    for k in (0, 5, 60, 900, V // 2):
        want = op.forward(l, u, temperature=0.8, top_k=k, top_p=0.9)
        got = op.forward(l, u, temperature=full(0.8), top_k=k, top_p=full(0.9), min_p=full(math.nan))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k
        want = op.forward(l, u, temperature=0.8, top_k=k, min_p=0.01)
        got = op.forward(l, u, temperature=0.8, top_k=k, top_p=full(math.nan), min_p=full(0.01))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k
        want = op.forward(l, u, temperature=0.0, top_k=k)
        got = op.forward(l, u, temperature=full(math.nan), top_k=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k
        want = op.forward(l, full(0.0), top_k=k)
        got = op.forward(l, full(math.nan), top_k=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k


def test_negative_min_p_restricts_nothing():
    from mgpt_amd.sampling import Sampler
    for V in (500, 20000):
        l, u = inputs(8, V, "f32")
        for k in (0, 60):
            want = Sampler(V).forward(l, u, top_k=k)
            got = Sampler(V).forward(l, u, top_k=k, min_p=torch.full((8,), -1.0, device="cuda"))
            assert torch.equal(got[0], want[0])


def test_more_rows_than_a_launch_takes():
    """2^22 blocks of 1024 threads are more than a grid holds: it ran those past them alone."""
    B = (1 << 22) + 1000
    gen = torch.Generator(device="cuda").manual_seed(1)
    l = torch.randn(B, 3, generator=gen, device="cuda").bfloat16()
    check(l, torch.rand(B, generator=gen, device="cuda"), T=torch.rand(B, generator=gen, device="cuda"), k=2, p=0.9)
