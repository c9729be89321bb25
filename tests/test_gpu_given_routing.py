"""MoELayer.forward_routed with routings that a router does not make: the same expert several times for a token, all
tokens to one, ids out of range, weights of any sign, in every type of weights.  Against the experts in 64 bits: each
term has the layer's own bar (test_gpu_layer_routing.py) of its size, which the terms' sum may be far below."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_layer_routing import BAR, Case  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act,weights", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "fp8"), ("f32", "fp8"), ("f32", "bf16"),
                                         ("bf16", "i8"), ("f32", "i8")])
@pytest.mark.parametrize("E,k,C", [(8, 4, 128), (64, 8, 256), (80, 2, 192)])
def test_any_ids(E, k, C, act, weights):
    c = Case(C, 256, E, k, act, weights)
    for N in (1, 20, 64, 700):
        gen = torch.Generator(device="cuda").manual_seed(N)
        x = c.x(N)
        w = torch.randn(N, k, generator=gen, device="cuda")
        few = torch.randint(0, 3, (N, k), generator=gen, device="cuda", dtype=torch.int32)
        one = torch.full((N, k), E - 1, device="cuda", dtype=torch.int32)
        out = torch.randint(-2, E + 3, (N, k), generator=gen, device="cuda", dtype=torch.int32)
        for idx in (few, one, out):
            y = c.op.forward_routed(x, idx, w)
            valid = (idx >= 0) & (idx < E)
            e, v = torch.where(valid, idx, torch.zeros_like(idx)).long(), torch.where(valid, w, torch.zeros_like(w)).double()
            terms = [c.experts(x.double(), e[:, j:j + 1], v[:, j:j + 1]) for j in range(k)]
            size = torch.stack([t.norm() for t in terms]).sum()
            assert (y.double() - sum(terms)).norm() <= BAR[weights] * size, (N, idx is few, idx is one)
            assert torch.equal(y, c.op.forward_routed(x, idx, w))
