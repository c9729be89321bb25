"""mgpt_norm_forward / mgpt_norm_backward against the formulas in 64 bits where each
of their kernels runs: rows of 1 to 16 waves, outputs that are stored past the caches,
groups split over blocks and whole ones, gains left out, offsets past 32 bits.

Tolerances, u = 2^-24, as in test_gpu_norm: a value formed by k roundings of terms that
sum to A in magnitude is within k u A; out 64, y and its rms 128, dx and dh 256 (two
means over a row); bf16 outputs another half step, 2^-8 of them.  A column sum adds its
own roundings to its terms' 256: here a stream has at most 33 rows that are not zero, a block
4 streams, a quarter of a wave's blocks is 8, 16 waves and 3 groups: under 128.
Each group's first and last rows and some others have upstream gradients 30 times as
large, so that one of them left out of a column sum shows.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
EPS = 1e-5
ALL = ("post", "gate", "pre")


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()
    yield
    torch.cuda.empty_cache()


def inputs(N, C, G, act, seed=7):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.float32 if act == "f32" else torch.bfloat16
    rows = {k: (torch.randn(N, C, generator=gen, device="cuda") * s).to(dt)
            for k, s in (("x", 2.0), ("h", 0.7), ("dout", 1.0), ("dy", 1.0))}
    edges = torch.cat([torch.arange(0, N, N // G), torch.arange(N // G - 1, N, N // G), torch.arange(0, N, N // 7 + 1)])
    edges = edges.unique().cuda()
    for k in ("dout", "dy"):
        rows[k][edges] *= 30
    gains = {"post": 1 + 0.2 * torch.randn(C, generator=gen, device="cuda"),
             "gate": torch.randn(G, C, generator=gen, device="cuda"),
             "pre": 1 + 0.2 * torch.randn(C, generator=gen, device="cuda")}
    return rows, gains


def reference(rows, gains, G, s, use, dout):
    """{name: (value, magnitude of its terms, roundings)} in 64 bits, all at once."""
    x, h, do, dy = (rows[k].double() for k in ("x", "h", "dout", "dy"))
    N, C = x.shape
    ref = {}
    post = gains["post"].double() if "post" in use else torch.ones(C, dtype=torch.float64, device="cuda")
    gate = gains["gate"].double().repeat_interleave(N // G, 0) if "gate" in use else torch.ones_like(x)
    n = h
    if "post" in use:
        rh = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        n = h * rh
        ref["rh"] = (rh[:, 0], rh[:, 0], 64)
    o = s * x + gate * n * post
    ao = (s * x).abs() + (gate * n * post).abs()
    ref["out"] = (o, ao, 64)
    d, ad = (do, do.abs()) if dout else (torch.zeros_like(x), torch.zeros_like(x))
    if "pre" in use:
        pre = gains["pre"].double()
        ro = 1 / torch.sqrt((o * o).mean(1, keepdim=True) + EPS)
        more = 1 + (ao * ao).mean(1, keepdim=True) * ro ** 2   # the roundings of o in its mean
        z, az = o * ro, ao * ro * more
        q = dy * pre
        ref["ro"] = (ro[:, 0], (ro * more)[:, 0], 128)
        ref["y"] = (z * pre, az * pre.abs(), 128)
        ref["dpre"] = ((dy * z).sum(0), (dy.abs() * az).sum(0), 384)
        d = d + ro * (q - z * (q * z).mean(1, keepdim=True))
        ad = ad + ro * more * (q.abs() + az * (q.abs() * az).mean(1, keepdim=True))
    ref["dx"] = (s * d, s * ad, 256)
    w, aw = d * gate * post, ad * (gate * post).abs()
    ref["dh"] = (w, aw, 256)
    if "post" in use:
        ref["dh"] = (rh * (w - n * (w * n).mean(1, keepdim=True)),
                     rh * (aw + n.abs() * (aw * n.abs()).mean(1, keepdim=True)), 256)
        ref["dpost"] = ((d * gate * n).sum(0), (ad * (gate * n).abs()).sum(0), 384)
    if "gate" in use:
        ref["dgate"] = ((d * n * post).view(G, -1, C).sum(1), (ad * (n * post).abs()).view(G, -1, C).sum(1), 384)
    return ref


def run(rows, gains, s, use, act, dout):
    from mgpt_amd.norm import ResidualNorm
    op = ResidualNorm(rows["x"].shape[1], act=act, eps=EPS, residual_scale=s)
    g = {k if k == "gate" else "gamma_" + k: v if k in use else None for k, v in gains.items()}
    out, y, rh, ro = op.forward(rows["x"], rows["h"], **g)
    dx, dh, dpost, dgate, dpre = op.backward(rows["x"], rows["h"], rows["dout"] if dout else None,
                                             rows["dy"] if "pre" in use else None, rh, ro, **g)
    got = {"out": out, "y": y, "rh": rh, "ro": ro, "dx": dx, "dh": dh, "dpost": dpost, "dgate": dgate, "dpre": dpre}
    return {k: v for k, v in got.items() if v is not None}


def check(got, ref, act):
    assert set(got) == set(ref)
    for k, (want, amp, roundings) in ref.items():
        tol = roundings * U * amp
        if act == "bf16" and k in ("out", "y", "dx", "dh"):
            tol = tol + 2.0 ** -8 * (want.abs() + tol)
        err = (got[k].double().view(want.shape) - want).abs()
        assert (err <= tol).all(), (k, float((err / tol.clamp(min=1e-300)).max()), int((err > tol).sum()))


def compare(N, C, G, act, use=ALL, s=0.7, dout=True):
    print(N, C, G, act, use, dout, flush=True)
    rows, gains = inputs(N, C, G, act)
    check(run(rows, gains, s, use, act, dout), reference(rows, gains, G, s, use, dout), act)


# dx and dh of 128 MB and more together in bf16, as much with half the rows in fp32; 1 to
# 16 waves a row in the backward
LONG = [(66600, 504, 1), (33600, 1000, 3), (16400, 2048, 2), (8202, 4096, 1), (4106, 8184, 1)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,G", LONG)
def test_outputs_past_the_caches(N, C, G, act):
    compare(N if act == "bf16" else N // 2 // G * G, C, G, act)


# both norms and dout: groups of 8 rows and more, and whole groups of fewer
WIDE = [(40, 4096, 2), (42, 8192, 2), (24, 16384, 1), (30, 8200, 3), (5, 1000, 1), (6, 2000, 1)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,G", WIDE)
def test_wide_rows(N, C, G, act):
    compare(N, C, G, act)


# a gain or dout left out: the engine's own block has the norm behind the sum alone, the
# last block no dout
PARTLY = [(20, 2048, 2), (20, 4096, 2), (18, 8192, 2), (600, 136, 2), (64, 1024, 1)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("use,dout", [(("pre",), True), (("gate", "pre"), True), (ALL, False), (("post", "gate"), True)])
@pytest.mark.parametrize("N,C,G", PARTLY)
def test_blocks_without_all_gains(N, C, G, use, dout, act):
    compare(N, C, G if "gate" in use else 1, act, use, dout=dout)


def test_the_far_end_of_rows_past_4_gib():
    """Zero rows but for the last 40: those, and the column sums, which have no other
    terms."""
    from mgpt_amd.norm import ResidualNorm
    N, C, last = 280001, 8192, slice(280001 - 40, 280001)
    rows, gains = inputs(40, C, 1, "bf16")
    far = {}
    for k, v in rows.items():
        far[k] = torch.zeros(N, C, dtype=v.dtype, device="cuda")
        far[k][last] = v
    got = run(far, gains, 0.7, ALL, "bf16", True)
    for k in ("out", "y", "dx", "dh"):
        assert not got[k][:64].any() and not got[k][N // 2:N // 2 + 64].any()
    got = {k: v[last] if v.shape[0] == N else v for k, v in got.items()}
    check(got, reference(rows, gains, 1, 0.7, ALL, True), "bf16")
