"""Routing, the integer linear layer and sampling with sizes that 32 bits do not hold, or none at all: refused, or what
they mean."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def test_rows_past_32_bits():
    from mgpt_amd.linear8 import I8Linear
    from mgpt_amd.routing import ExpertRouting
    from mgpt_amd.sampling import Sampler
    N = (1 << 32) + 5
    x = torch.empty(N, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="rows"):
        Sampler(1, act="bf16").forward(x, torch.empty(N, dtype=torch.float32, device="cuda"))
    op = I8Linear(1, 1)
    op.load_quantized(torch.ones(1, 1, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    with pytest.raises(ValueError, match="rows"):
        op.forward(x)
    rule = ExpertRouting(1, 1, act="bf16")
    with pytest.raises(ValueError, match="rows"):
        rule.forward(x)
    idx = torch.empty(N, 1, dtype=torch.int32, device="cuda")
    w = torch.empty(N, 1, dtype=torch.float32, device="cuda")
    with pytest.raises(ValueError, match="rows"):
        rule.backward(x, idx, w, w)


def test_no_experts():
    from mgpt_amd import capi
    from mgpt_amd.routing import ExpertRouting
    with pytest.raises(capi.MoEError):
        ExpertRouting(0, 1).forward(torch.empty(4, 0, device="cuda"))


def test_top_k_of_any_size():
    from mgpt_amd.sampling import Sampler
    gen = torch.Generator(device="cuda").manual_seed(1)
    for V in (300, 20000):
        l, u = torch.randn(9, V, generator=gen, device="cuda"), torch.rand(9, generator=gen, device="cuda")
        op = Sampler(V)
        want = op.forward(l, u)
        for k in (0, -1, V, V + 1, 2 ** 31, 2 ** 32 + 3, -(2 ** 32) + 3, 2 ** 70):
            got = op.forward(l, u, top_k=k)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k


def test_more_tokens_than_a_grid_holds():
    import ctypes
    from mgpt_amd import capi
    from mgpt_amd.moe import MoELayer
    for weights, k in (("bf16", 2), ("i8", 4)):
        L = MoELayer(64, 64, 4, k, act="bf16", weights=weights)
        r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
        L.load_parameters([r(64, 4), r(4)] + 4 * [r(64, 64), r(64), r(64, 64), r(64), r(64, 64), r(64)])
        x, y, ws = (ctypes.c_void_p(a << 20) for a in (1, 1 << 30, 1 << 31))     # never read: refused before
        lib = capi.lib()
        for n, status in ((1 << 26, capi.MGPT_ERR_UNSUPPORTED), ((1 << 26) - 1, capi.MGPT_ERR_WORKSPACE_TOO_SMALL)):
            assert lib.mgpt_moe_forward(L._h, x, y, n, ws, 0, None) == status
            assert lib.mgpt_moe_forward_routed(L._h, x, x, x, y, n, ws, 0, None) == status
    L = MoELayer(64, 64, 4, 2, act="bf16")
    L.load_parameters([r(64, 4), r(4)] + 4 * [r(64, 64), r(64), r(64, 64), r(64), r(64, 64), r(64)])
    assert lib.mgpt_moe_forward_train(L._h, x, y, 1 << 25, ws, 0, None) == capi.MGPT_ERR_UNSUPPORTED
