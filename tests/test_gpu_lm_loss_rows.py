"""The language model's loss where its logits are known exactly: what the sums and
probabilities of a row lose by themselves, for rows whose logits are far from 0.

Row n's logits are a_n + b_v, a_n = n / 2 from 60 on and b_v = v / 8: x holds a_n in
its first column, W ones, and every product and sum of the logits is exact in fp32
and in bf16.  u = 2^-24.
  An exponential of z - s: its argument's multiple of log2 e is rounded (u of it) and
  log2 e itself (u), so 2 u |z - s|; the hardware's exp2 is off by a unit in the last
  place (2 u).  What a common rounding of s log2 e takes is put back by a factor of
  3 roundings.
  A row's sum of 8 of them adds 7 u, its logarithm, at most log 8, 2 units (9 u), and
  lse is rounded once more: u |lse| + (2 range + 2 + 3 + 7 + 9) u.
  A probability from a given lse: (2 |z - lse| + 2 + 3) u, and u for its product with
  the upstream gradient; the target's difference u of itself.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
N, C, V = 70, 64, 8


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


def exact_logits(act):
    """(x, W, b, t) and the logits in 64 bits."""
    dt = torch.float32 if act == "f32" else torch.bfloat16
    a = 60 + torch.arange(N, dtype=torch.float64) / 2
    b = torch.arange(V, dtype=torch.float64) / 8
    x, W = torch.zeros(N, C, dtype=torch.float64), torch.zeros(V, C, dtype=torch.float64)
    x[:, 0] = a
    W[:, 0] = 1
    W[torch.arange(V), 1 + torch.arange(V)] = 1   # x is 0 there: d shows in dx
    t = torch.arange(N, dtype=torch.int32) % V
    assert torch.equal(x.to(dt).double(), x)
    return x.to(dt).cuda(), W.to(dt).cuda(), b.float().cuda(), t.cuda(), (a[:, None] + b).cuda()


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_log_sum_exp(act):
    from mgpt_amd.loss import LMLoss
    x, W, b, t, z = exact_logits(act)
    loss, lse, mean = LMLoss(C, V, act=act).forward(x, W, t, bias=b)
    want = torch.logsumexp(z, 1)
    err = (lse.double() - want).abs()
    tol = U * want + (2 * (V - 1) / 8 + 21) * U
    assert (err <= tol).all(), (float((err / tol).max()), int((err > tol).sum()))


def reference(z, lse, t):
    """d of the sum of the rows' losses, from lse as it is held, and its tolerance."""
    p = (z - lse.double()[:, None]).exp()
    d = p - torch.nn.functional.one_hot(t.long(), V)
    return d, (p * (2 * (z - lse.double()[:, None]).abs() + 6) + d.abs()) * U


def test_gradients_of_the_logits():
    """fp32: d passes through dx whole, times ones (one more u for the product)."""
    from mgpt_amd.loss import LMLoss
    x, W, b, t, z = exact_logits("f32")
    lse = torch.logsumexp(z, 1).float()
    want, tol = reference(z, lse, t)
    dx, _, _ = LMLoss(C, V, act="f32").backward(x, W, t, lse, bias=b, dloss=torch.ones(N, device="cuda"))
    err = (dx[:, 1:1 + V].double() - want).abs()
    tol = tol + U * want.abs()
    assert (err <= tol).all(), (float((err / tol).max()), int((err > tol).sum()))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_gradient_of_the_bias_of_one_row(act):
    """A single row's d is its dbias, in fp32 for either type."""
    from mgpt_amd.loss import LMLoss
    x, W, b, t, z = exact_logits(act)
    lse = torch.logsumexp(z, 1).float()
    want, tol = reference(z, lse, t)
    op = LMLoss(C, V, act=act)
    got = torch.stack([op.backward(x[n:n + 1], W, t[n:n + 1], lse[n:n + 1], bias=b)[2] for n in range(N)])
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), int((err > tol).sum()))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_an_infinite_upstream_gradient(act):
    """(p - [v = t]) times it: infinite, and of the sign of the difference."""
    from mgpt_amd.loss import LMLoss
    x, W, b, t, z = exact_logits(act)
    lse = torch.logsumexp(z, 1).float()
    op = LMLoss(C, V, act=act)
    for g in (float("inf"), float("-inf")):
        for n in (0, 5, 69):
            dloss = torch.full((1,), g, device="cuda")
            _, _, db = op.backward(x[n:n + 1], W, t[n:n + 1], lse[n:n + 1], bias=b, dloss=dloss)
            want = torch.full((V,), g, device="cuda")
            want[int(t[n])] = -g
            assert torch.equal(db, want), (g, n, db)


FAR = [1e4, 3e6, 1e9, 1e10, 1e20, 1e30, 3e38]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_rows_of_far_logits(act, sign):
    """Rows whose logits are all one number, up to the largest and down to the lowest
    (masked ones): lse is within its rounding of it, and the probabilities from a
    given lse are those of its difference from the logits."""
    from mgpt_amd.loss import LMLoss
    dt = torch.float32 if act == "f32" else torch.bfloat16
    n = len(FAR)
    x, W = torch.zeros(n, C, dtype=dt, device="cuda"), torch.zeros(V, C, dtype=dt, device="cuda")
    x[:, 0] = sign * torch.tensor(FAR)
    W[:, 0] = 1
    a = x[:, 0].to(torch.bfloat16)   # a single part of a split product
    x[:, 0] = a
    t = torch.arange(n, dtype=torch.int32, device="cuda")
    b = torch.zeros(V, device="cuda")
    z = a.double()[:, None].expand(n, V)
    op = LMLoss(C, V, act=act)
    loss, lse, mean = op.forward(x, W, t, bias=b)
    want = torch.logsumexp(z, 1)
    assert ((lse.double() - want).abs() <= U * want.abs() + 21 * U).all(), lse
    assert ((loss.double() - want + z[:, 0]).abs() <= U * want.abs() + 22 * U).all(), loss
    given = want.float()
    d, tol = reference(z, given, t)
    got = torch.stack([op.backward(x[i:i + 1], W, t[i:i + 1], given[i:i + 1], bias=b)[2] for i in range(n)])
    assert ((got.double() - d).abs() <= tol).all(), got
