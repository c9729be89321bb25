"""mgpt_lm_loss_forward / mgpt_lm_loss_backward against 64 bits, with test_gpu_lm_loss's
tolerances, at shapes whose products take 64 x 128 tiles in every way: logits and their
gradients over many tiles and over few, few rows, products with 5 slots and 9 that are added
up, and gradients of few rows and very wide ones, stored whole, by odd rows too."""
import pytest

from test_gpu_lm_loss import check, inputs, reference, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


# logits: many tiles, several rows of them, and few
LOGITS = {"bf16": [(141, 8, 17129), (190, 441, 33000), (2, 64, 22713)],
          "f32": [(289, 8, 11842), (156, 320, 18358), (8, 64, 19456)]}
# fp32 parts of a split contraction
PARTS = [(1142, 2240, 132), (4429, 67, 480), (1580, 101, 9460)]
# widths past 16384 columns: dx of few rows, dW of a small vocabulary
WIDE = [(2, 16456, 2), (3, 33560, 5), (5, 17877, 3), (1, 51135, 1), (40, 19512, 33), (60, 20379, 7), (3, 36211, 2),
        (7, 48712, 4)]


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("act,N,C,V", [(a, *s) for a in LOGITS for s in LOGITS[a]])
def test_logits(act, N, C, V, bias):
    print(N, C, V, act, bias, flush=True)
    x, W, b, t = inputs(N, C, V, act, bias=bias)
    check(run(x, W, b, t, act), reference(x, W, b, t))


@pytest.mark.parametrize("N,C,V", PARTS)
def test_parts_in_fp32(N, C, V):
    print(N, C, V, flush=True)
    x, W, b, t = inputs(N, C, V, "f32")
    check(run(x, W, b, t, "f32"), reference(x, W, b, t))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,V", WIDE)
def test_few_rows_of_many_columns(N, C, V, act):
    print(N, C, V, act, flush=True)
    x, W, b, t = inputs(N, C, V, act)
    check(run(x, W, b, t, act), reference(x, W, b, t))
