"""Places of a routing that no expert takes: ids out of range in MoELayer.forward_routed and weights of 0.  They count
for nothing: not in y, whatever is in x, and not in the experts' counts.  Bars as in test_gpu_layer_routing.py: of an output the bar is on
each term's size, so that on their sum's it is at most that of the sizes' sum, which the sum may be far below (three
terms of one token under fp8 weights)."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_layer_routing import BAR, Case  # noqa: E402

INF, NAN = float("inf"), float("nan")
KINDS = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "fp8"), ("f32", "fp8"), ("f32", "bf16"), ("bf16", "i8"), ("f32", "i8")]


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def sizes(c, x, idx, w):
    """The sum over the places of their terms' norms."""
    return sum(c.experts(x.double(), idx[:, j:j + 1], w[:, j:j + 1].double()).norm() for j in range(idx.shape[1]))


@pytest.mark.parametrize("act,weights", KINDS)
@pytest.mark.parametrize("E,k,C", [(8, 4, 128), (8, 2, 64), (64, 8, 256), (80, 2, 192), (6, 1, 100)])
def test_ids_out_of_range_and_weights_of_zero(E, k, C, act, weights):
    c = Case(C, 128, E, k, act, weights)
    for N in (1, 20, 64, 300, 1500):
        gen = torch.Generator(device="cuda").manual_seed(N)
        x = c.x(N)
        idx = torch.rand(N, E, generator=gen, device="cuda").topk(k, 1)[1].int()
        w = torch.rand(N, k, generator=gen, device="cuda") + 0.1
        none = torch.rand(N, k, generator=gen, device="cuda") < 0.3
        none[::3] = True                     # tokens of no expert at all
        x[::3, 5] = NAN
        x[::6, 7] = INF
        out = torch.where(none, torch.where(idx % 2 == 0, -1, E + 3).int(), idx)
        zero = torch.where(none, torch.zeros_like(w), w)
        y = c.op.forward_routed(x, out, w)
        r = c.op.routing()
        assert torch.equal(r["counts"].long(), torch.bincount(idx[~none].long(), minlength=E))
        assert (y[::3] == 0).all()
        live = torch.ones(N, dtype=torch.bool, device="cuda")
        live[::3] = False
        if live.any():
            want = c.experts(x[live].double(), torch.where(none, -1, idx)[live], w[live].double())
            assert (y[live].double() - want).norm() <= BAR[weights] * sizes(c, x[live], torch.where(none, -1, idx)[live], w[live])
        assert same(c.op.forward_routed(x, idx, zero), y)
        assert same(c.op.forward_routed(x, torch.full_like(idx, -1), w), torch.zeros_like(y))


def test_replayed_graph():
    c = Case(64, 96, 8, 2, "bf16", "i8")
    for N in (30, 500):
        x = c.x(N)
        idx = torch.zeros(N, 2, dtype=torch.int32, device="cuda")
        w = torch.ones(N, 2, device="cuda")
        c.op.forward_routed(x, idx, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = c.op.forward_routed(x, idx, w)
        for seed in (3, 4, 5):
            gen = torch.Generator(device="cuda").manual_seed(seed)
            idx.copy_(torch.randint(-4, 8, (N, 2), generator=gen, device="cuda", dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            assert torch.equal(got, c.op.forward_routed(x, idx, w))
            assert (got[(idx < 0).all(1)] == 0).all()
