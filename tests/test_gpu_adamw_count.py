"""The number of an AdamW optimizer's steps when it is held on the device: what
step_count says and sets there is what the next step, eager or replayed, counts
on from."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


def make(p, **kw):
    from mgpt_amd.optim import AdamW
    return AdamW([p], lr=1e-2, **kw)


def grads(n, count):
    gen = torch.Generator().manual_seed(4)
    return [torch.randn(n, generator=gen).cuda() for _ in range(count)]


@pytest.mark.parametrize("bits", [32, 8])
def test_training_goes_on_from_a_saved_state(bits):
    """Parameters, state and step_count of a run copied into an optimizer with its
    number on the device: the next steps have the run's bits."""
    gs = grads(700, 5)
    p = torch.ones(700, device="cuda")
    a = make(p, state_bits=bits)
    for g in gs[:3]:
        a.step([g])
    assert a.step_count == 3
    q = p.clone()
    b = make(q, state_bits=bits, device_step=True)
    b.state.copy_(a.state)
    b.step_count = a.step_count
    for g in gs[3:]:
        a.step([g])
        b.step([g])
        assert torch.equal(p, q) and torch.equal(a.state, b.state)
    assert a.step_count == b.step_count == 5


def test_replayed_steps_are_counted_and_a_captured_one_is_not():
    gs = grads(700, 4)
    p = torch.ones(700, device="cuda")
    q, g = p.clone(), torch.zeros(700, device="cuda")
    a, b = make(p), make(q, device_step=True)
    a.step([gs[0]])
    g.copy_(gs[0])
    b.step([g])
    assert b.step_count == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step([g])
    assert b.step_count == 1
    for i, gi in enumerate(gs[1:]):
        a.step([gi])
        g.copy_(gi)
        graph.replay()
        assert b.step_count == a.step_count == i + 2
        assert torch.equal(p, q)
    # the graph counts on from a number that is set
    a.step_count = b.step_count = 100
    a.step([gs[0]])
    g.copy_(gs[0])
    graph.replay()
    assert torch.equal(p, q) and b.step_count == 101


def test_a_refused_step_is_not_counted_on_the_device():
    from mgpt_amd.capi import MoEError
    p = torch.ones(300, device="cuda")
    opt = make(p, device_step=True)
    opt.step_count = 7
    opt.lr = float("nan")
    with pytest.raises(MoEError):
        opt.step([torch.ones(300, device="cuda")])
    assert opt.step_count == 7
