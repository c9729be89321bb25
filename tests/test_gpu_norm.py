"""mgpt_norm_forward / mgpt_norm_backward (mgpt_amd.norm.ResidualNorm) against
the formulas in 64 bits on the CPU, every gain present or left out, and the
backward against differences of the forward.

Tolerances: u = 2^-24.  A value formed by k fp32 roundings of terms that sum
to A in magnitude is within k u A.  A row's mean is at most 16 products and
sums a lane, 6 steps over a wave and 16 over a row's waves: under 64 roundings,
of which a reciprocal square root keeps half.  So out is within 64 u (|s x| +
|w|) and y within 128 u of its terms; the gradients of rows pass through two
such means (256 u), and a column sum adds at most N roundings of its terms
(256 + N) u.  In bf16 every output of that type adds half a step, 2^-8 of it (2^-9
of its power of two's double).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mgpt_amd import capi
    capi.lib()


def inputs(N, C, G, act, seed=3):
    rng = np.random.default_rng(seed)
    dt = torch.float32 if act == "f32" else torch.bfloat16
    rows = {k: torch.from_numpy(rng.standard_normal((N, C)) * s).to(dt)
            for k, s in (("x", 2.0), ("h", 0.7), ("dout", 1.0), ("dy", 1.0))}
    gains = {"post": torch.from_numpy(1 + 0.2 * rng.standard_normal(C)).float(),
             "gate": torch.from_numpy(rng.standard_normal((G, C))).float(),
             "pre": torch.from_numpy(1 + 0.2 * rng.standard_normal(C)).float()}
    return rows, gains


def reference(rows, gains, G, s, use, dout=True):
    """{name: (value, magnitude of its terms, roundings)} in 64 bits."""
    x, h, do_, dy = (rows[k].double().numpy() for k in ("x", "h", "dout", "dy"))
    N, C = x.shape
    one = np.ones(C)
    post = gains["post"].double().numpy() if "post" in use else one
    pre = gains["pre"].double().numpy() if "pre" in use else one
    gate = np.repeat(gains["gate"].double().numpy(), N // G, 0) if "gate" in use else np.ones((N, C))
    rh = 1 / np.sqrt((h * h).mean(1, keepdims=True) + EPS) if "post" in use else np.ones((N, 1))
    n = h * rh
    w = gate * n * post
    o, ao = s * x + w, np.abs(s * x) + np.abs(w)
    out = {"out": (o, ao, 64)}
    if "post" in use:
        out["rh"] = (rh[:, 0], rh[:, 0], 64)
    d = do_ if dout else np.zeros_like(x)
    ad = np.abs(d)
    if "pre" in use:
        ro = 1 / np.sqrt((o * o).mean(1, keepdims=True) + EPS)
        # the terms of o, not o itself, carry its roundings into the mean
        ro_amp = (ao * ao).mean(1, keepdims=True) * ro ** 2
        z, az = o * ro, ao * ro * (1 + ro_amp)
        out["ro"] = (ro[:, 0], (ro * (1 + ro_amp))[:, 0], 128)
        out["y"] = (z * pre, az * np.abs(pre), 128)
        q = dy * pre
        d = d + ro * (q - z * (q * z).mean(1, keepdims=True))
        ad = ad + ro * (1 + ro_amp) * (np.abs(q) + az * (np.abs(q) * az).mean(1, keepdims=True))
        out["dpre"] = ((dy * z).sum(0), (np.abs(dy) * az).sum(0), 256 + N)
    out["dx"] = (s * d, s * ad, 256)
    dn, adn = d * gate * post, ad * np.abs(gate * post)
    if "post" in use:
        out["dh"] = (rh * (dn - n * (dn * n).mean(1, keepdims=True)),
                     rh * (adn + np.abs(n) * (adn * np.abs(n)).mean(1, keepdims=True)), 256)
        out["dpost"] = ((d * gate * n).sum(0), (ad * np.abs(gate * n)).sum(0), 256 + N)
    else:
        out["dh"] = (dn, adn, 256)
    if "gate" in use:
        out["dgate"] = ((d * n * post).reshape(G, -1, C).sum(1), (ad * np.abs(n * post)).reshape(G, -1, C).sum(1),
                        256 + N)
    return out


def run(rows, gains, G, s, use, act, dout=True):
    from mgpt_amd.norm import ResidualNorm
    op = ResidualNorm(rows["x"].shape[1], act=act, eps=EPS, residual_scale=s)
    r = {k: v.cuda() for k, v in rows.items()}
    g = {"gamma_" + k if k != "gate" else k: gains[k].cuda() if k in use else None for k in gains}
    out, y, rh, ro = op.forward(r["x"], r["h"], **g)
    dx, dh, dpost, dgate, dpre = op.backward(r["x"], r["h"], r["dout"] if dout else None,
                                             r["dy"] if "pre" in use else None, rh, ro, **g)
    got = {"out": out, "y": y, "rh": rh, "ro": ro, "dx": dx, "dh": dh, "dpost": dpost, "dgate": dgate, "dpre": dpre}
    torch.cuda.synchronize()
    return {k: v for k, v in got.items() if v is not None}


def check(got, ref, act):
    assert set(got) == set(ref)
    for k, (want, amp, roundings) in ref.items():
        have = got[k].double().cpu().numpy().reshape(want.shape)
        tol = roundings * U * amp
        if act == "bf16" and k in ("out", "y", "dx", "dh"):
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
        err = np.abs(have - want)
        assert (err <= tol).all(), (k, float((err / np.maximum(tol, 1e-300)).max()))


ALL = ("post", "gate", "pre")
SHAPES = [(1, 1, 1), (1, 8, 1), (3, 7, 3), (5, 64, 1), (64, 2048, 1), (37, 1000, 1), (130, 513, 13), (33, 1032, 1),
          (96, 1024, 4), (3000, 72, 1500), (4100, 24, 2050), (9, 4096, 3), (7, 4100, 1), (5, 8192, 5), (3, 8200, 1),
          (2, 16384, 1), (1030, 256, 2)]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,G", SHAPES)
def test_forward_and_gradients(N, C, G, act):
    print(N, C, G, act, flush=True)
    rows, gains = inputs(N, C, G, act)
    check(run(rows, gains, G, 0.7, ALL, act), reference(rows, gains, G, 0.7, ALL), act)


@pytest.mark.parametrize("use", [(), ("post",), ("gate",), ("pre",), ("post", "gate"), ("post", "pre"), ("gate", "pre")])
@pytest.mark.parametrize("N,C,G", [(40, 200, 4), (11, 2056, 1), (6, 64, 6)])
def test_gains_left_out(N, C, G, use):
    rows, gains = inputs(N, C, G, "f32")
    check(run(rows, gains, G, 1.0, use, "f32"), reference(rows, gains, G, 1.0, use), "f32")
    if "pre" in use:
        check(run(rows, gains, G, 1.0, use, "f32", dout=False), reference(rows, gains, G, 1.0, use, False), "f32")


def test_rows_of_zeros_and_the_eps():
    rows, gains = inputs(8, 96, 1, "f32")
    rows["h"][2] = 0
    rows["x"][2] = 0
    rows["h"][5] = 0
    check(run(rows, gains, 1, 1.0, ALL, "f32"), reference(rows, gains, 1, 1.0, ALL), "f32")


def test_gradients_are_the_forwards_differences():
    """d(sum(out * dout + y * dy)) along random directions: central differences
    of the forward in 64 bits against the kernel's gradients.  With steps of
    1e-5 the difference's own error is under 1e-8 of the terms; the
    gradients' (256 + N) u of their terms is 1.7e-5 for N = 24."""
    N, C, G, s = 24, 40, 3, 0.6
    rows, gains = inputs(N, C, G, "f32")
    got = run(rows, gains, G, s, ALL, "f32")

    def value(r, g):
        ref = reference(r, g, G, s, ALL)
        return ref["out"][0], ref["y"][0]

    rng = np.random.default_rng(11)
    for name, grad in (("x", "dx"), ("h", "dh"), ("post", "dpost"), ("gate", "dgate"), ("pre", "dpre")):
        src = rows if name in rows else gains
        v = torch.from_numpy(rng.standard_normal(tuple(src[name].shape)))
        ends = []
        for sign in (1, -1):
            moved = {k: t.double() for k, t in src.items()}
            moved[name] = moved[name] + sign * 1e-5 * v
            r, g = (moved, {k: t.double() for k, t in gains.items()}) if src is rows else (rows, moved)
            ends.append(value(r, g))
        dout, dy = rows["dout"].double().numpy(), rows["dy"].double().numpy()
        diff = ((ends[0][0] - ends[1][0]) * dout + (ends[0][1] - ends[1][1]) * dy).sum() / 2e-5
        along = (got[grad].double().cpu().numpy().reshape(v.shape) * v.numpy())
        assert abs(diff - along.sum()) <= 3e-5 * np.abs(along).sum(), (name, diff, along.sum())


def test_same_bits_again_on_another_stream_and_in_a_graph():
    from mgpt_amd.norm import ResidualNorm
    rows, gains = inputs(200, 1024, 2, "bf16")
    first = run(rows, gains, 2, 0.5, ALL, "bf16")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = run(rows, gains, 2, 0.5, ALL, "bf16")
    for k in first:
        assert torch.equal(first[k], again[k]), k
    op = ResidualNorm(1024, act="bf16", eps=EPS, residual_scale=0.5)
    r = {k: v.cuda() for k, v in rows.items()}
    g = dict(gamma_post=gains["post"].cuda(), gate=gains["gate"].cuda(), gamma_pre=gains["pre"].cuda())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, y, rh, ro = op.forward(r["x"], r["h"], **g)
        grads = op.backward(r["x"], r["h"], r["dout"], r["dy"], rh, ro, **g)
    for _ in range(3):
        for t in (out, y, *grads):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        have = dict(zip(("out", "y", "dx", "dh", "dpost", "dgate", "dpre"), (out, y, *grads)))
        for k, t in have.items():
            assert torch.equal(first[k], t), k
        run(rows, gains, 2, 1.0, ALL, "bf16")


def test_no_tokens():
    from mgpt_amd.norm import ResidualNorm
    op = ResidualNorm(32, act="f32")
    e = torch.empty(0, 32, device="cuda")
    g = dict(gamma_post=torch.ones(32, device="cuda"), gate=torch.ones(32, device="cuda"),
             gamma_pre=torch.ones(32, device="cuda"))
    out, y, rh, ro = op.forward(e, e, **g)
    dx, dh, *gr = op.backward(e, e, e, e, rh, ro, **g)
    assert out.shape == (0, 32) and dx.shape == (0, 32)
    assert all((t == 0).all() for t in gr)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("N,C,G", [(9, 72, 1), (13, 1032, 1), (66, 520, 2)])
def test_an_infinity_stays_where_the_formulas_put_it(N, C, G, act):
    """An infinite dy in a group's last row: dgamma_pre is infinite in its column
    alone, dx of the row infinite (NaN in that column: inf - inf) and every other
    row's results are those without it."""
    rows, gains = inputs(N, C, G, act)
    clean = run(rows, gains, G, 0.7, ALL, act)
    rows["dy"][N - 1, 3] = float("inf")
    got = run(rows, gains, G, 0.7, ALL, act)
    last = torch.arange(N) == N - 1
    for k in ("dx", "dh"):
        assert torch.equal(got[k].reshape(N, C).cpu()[~last], clean[k].reshape(N, C).cpu()[~last]), k
    column = torch.arange(C) == 3
    dpre = got["dpre"].cpu().flatten()
    assert dpre[3].isinf() and torch.equal(dpre[~column], clean["dpre"].cpu().flatten()[~column])
    dx = got["dx"].reshape(N, C).cpu()[N - 1]
    assert dx[3].isnan() and dx[~column].isinf().all()
