"""The training step's operators over no tokens write their zeros to outputs that
lie at any element, as they do for some tokens, and to nothing beside them."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


class Output:
    """n sevens, `off` elements into a buffer of them."""

    def __init__(self, n, off, dtype=torch.float32):
        self.n, self.off = n, off
        self.buf = torch.full((n + off + 4,), 7.0, dtype=dtype, device="cuda")
        self.ptr = self.buf[off:].data_ptr()

    def zeroed(self):
        end = self.off + self.n
        return (self.buf[:self.off] == 7).all() and (self.buf[end:] == 7).all() and not self.buf[self.off:end].any()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("C,V", [(7, 9), (1, 1), (300, 33), (64, 20000)])
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_loss(act, C, V, off):
    from mgpt_amd import capi
    cfg = capi.LMLossConfig(C, V, capi.DTYPE_F32 if act == "f32" else capi.DTYPE_BF16)
    mean, db = Output(2, off), Output(V, off)
    dW = Output(V * C, off, torch.float32 if act == "f32" else torch.bfloat16)
    st = capi.stream(dW.buf.device)
    capi.check(capi.lib().mgpt_lm_loss_forward(ctypes.byref(cfg), None, None, None, None, None, None, mean.ptr, 0, None,
                                               0, st))
    capi.check(capi.lib().mgpt_lm_loss_backward(ctypes.byref(cfg), *[None] * 8, dW.ptr, db.ptr, 0, None, 0, st))
    assert mean.zeroed() and dW.zeroed() and db.zeroed()


@pytest.mark.parametrize("C,G", [(1, 1), (2, 1), (7, 5), (2048, 3)])
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_norms(C, G, off):
    from mgpt_amd import capi
    cfg = capi.NormConfig(C, capi.DTYPE_BF16, G, 1e-5, 1.0)
    gains = torch.ones(G * C, device="cuda")
    post, gate, pre = Output(C, off), Output(G * C, off), Output(C, off)
    capi.check(capi.lib().mgpt_norm_backward(ctypes.byref(cfg), None, None, *[gains.data_ptr()] * 3, *[None] * 6,
                                             post.ptr, gate.ptr, pre.ptr, 0, None, 0, capi.stream(gains.device)))
    assert post.zeroed() and gate.zeroed() and pre.zeroed()
